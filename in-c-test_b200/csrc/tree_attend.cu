// tree_attend.cu -- attention of a tree of drafted tokens over the latent
// cache (tree_attend.cuh has the formula and the work decomposition).
#include <atomic>
#include <cmath>

#include "attend_host.cuh"
#include "pdl.cuh"
#include "prof.cuh"
#include "sm100.cuh"
#include "tree_attend.cuh"

namespace kvl {

// ------------------------------------------------------------------ any shape
// One CTA per (head, node); online softmax in fp32 over chunks of 1024 rows.
// Runs for shapes other than 16 heads x 512 x 64.  A row that the node does
// not see is never read, so nothing in it can reach the result.  It is there to
// be right for every shape, not fast: a thread computes the score of one row on
// the CUDA cores (neighbouring threads read a row apart), and every node
// and head reads the cache anew.  16 heads x 256 x 64, 8 sequences of 2048 rows, 8
// nodes: 3190 us (Q8 3290) for 2.4 GFLOP and 11 MB, 16 x 512 x 32: 4580 (5760), 2
// heads x 64 x 8: 390 (220).
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
constexpr uint32_t kUnit = 4 * kBox;        // half a tile's latents: 64 rows x 256 dims

// Shared memory holds three key tiles: while the scores of tile g + 1 run, tile g
// waits for its P.V and tile g + 2 is on its way.  For that the query's latents
// lie in tensor memory (with the whole query in shared memory and two tiles,
// scores and P.V of a tile in turn, a tile took 3420 cycles, of which the tensor
// core worked about 1750).
constexpr int kUnits = 6;
constexpr uint32_t OFF_R = kUnits * kUnit;  // ropes of two tiles, until their scores are done;
                                            // Q8: then the second part of their weights
constexpr uint32_t OFF_P = OFF_R + 2 * kBox;
constexpr uint32_t OFF_QR = OFF_P + kBox;   // the query's rope box
constexpr uint32_t OFF_BAR = OFF_QR + kBox;

// Tensor memory, 512 columns x 128 lanes:
//   O       64 rows x 512, weight-stationary layout, 256 columns: dims [256 i,
//           256 i + 128) in columns [128 i, 128 i + 128) of lanes 0-63, the next
//           128 dims in lanes 64-127
//   scores  plain M = 64 layout: row r in lane 32 (r / 16) + r % 16, the other
//           half of the lanes free for a second matrix.  A row of A meets the D
//           of its own lane, so the even query boxes (lanes + 0) and the odd ones
//           (lanes + 16) give two partial sums, which the softmax adds.  bf16:
//           two buffers of 64 columns.  Q8: one, and 64 columns for the rope's
//           part, which the row scale does not touch
//   query   eight boxes of 64 dims, two to 32 columns
constexpr uint32_t kColS = 256, kColRope = kColS + 64, kColQ = kColS + 128;
constexpr uint32_t kOddLanes = 16u << 16;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kU16 = kUnit / 16, kB16 = kBox / 16;  // in units of a matrix descriptor
// Row scales of the tiles between their conversion and their softmax.  A tile's
// place in the ring of latents may have been the query's three steps before,
// which is copied as soon as the scores of the last item are done: then the
// third tile of an item is converted while the softmax has still to read the
// scales of the last item's last one, so four sets, not three.
constexpr int kScaleRing = 4;

constexpr int kSoftThreads = 256;    // warps 4-11: softmax and epilogue
constexpr int kConvertWarp = 12;       // Q8: warps 12-27 load and convert the latents,
constexpr int kConvertThreads = 256;   // 256 threads a CTA's even tiles, 256 the odd ones
template <bool Q8>
constexpr int threads() { return 128 + kSoftThreads + (Q8 ? 2 * kConvertThreads : 0); }

constexpr uint32_t kSteps = 8;  // of the ring that have barriers of their own
__device__ __forceinline__ uint32_t step_phase(uint32_t j) { return (j / kSteps) & 1; }

struct Bars {
  // of step j's unit h: [h][j % 8], phase j / 8.  full: its bytes are there (bf16,
  // unit 1: and the tile's rope); done: its half of the P.V (its copy to tensor
  // memory) is, so its place is free (Q8, unit 1: and the rope's place, where the
  // weights' second part lay; bf16: that is free once the scores are)
  uint64_t full[2][kSteps], done[2][kSteps];
  uint64_t r_full[2];              // Q8: the rope of tile g is there: [g % 2], phase g / 2
  uint64_t qr_full, q_done;        // q_done: the item's last scores are done
  uint64_t s_full[2], s_empty[2];  // of tile g: [g % 2], phase g / 2
  uint64_t p_full, o_empty, drain[2];
  uint32_t tmem_base;
  int abort;
  uint32_t nonfinite[8];
  uint32_t cleared[2][kTreeGroup][2];  // [tile % 2][node][key half]: rows cleared that the node sees
  float red[2][2][kTreeRows];  // row maxima or sums of the two key halves, alternate exchanges
  float alpha[kTreeRows];
};
typedef float Scales[kScaleRing][kTreeKeys];  // Q8, behind Bars: row scales of the tiles in flight
template <bool Q8>
constexpr uint32_t smem_bytes() { return OFF_BAR + sizeof(Bars) + (Q8 ? sizeof(Scales) : 0); }
static_assert(smem_bytes<false>() <= 232448 && smem_bytes<true>() <= 232448, "shared memory budget");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed pairs of fp32: one instruction for two operations.
__device__ __forceinline__ uint64_t pair_bits(float2 a) { return *reinterpret_cast<const uint64_t *>(&a); }
__device__ __forceinline__ float2 pair_of(uint64_t a) { return *reinterpret_cast<const float2 *>(&a); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return pair_of(d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return pair_of(d);
}

// Matrix descriptor of a SW128 operand from its low word; the high word (8-row
// groups 1024 bytes apart) is the same for all of them.
__device__ __forceinline__ uint64_t desc_of(uint32_t lo) {
  constexpr uint32_t hi = (1024 >> 4) | (1u << 14) | (LAYOUT_SW128 << 29);
  return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t lbo_bytes) {
  return saddr >> 4 | (lbo_bytes >> 4) << 16;
}

// Sixteen bf16, in one store where they are aligned to 32 bytes.
__device__ __forceinline__ void store_bf16x16(uint16_t *dst, bool aligned, const float (&o)[16]) {
  uint32_t v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = pack_bf16(o[2 * i], o[2 * i + 1]);
  if (aligned) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4 *>(dst)[0] = make_uint4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<uint4 *>(dst)[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// 32 bytes in one load where they are aligned to it.
__device__ __forceinline__ void load_32(const int8_t *src, bool aligned, uint4 &a, uint4 &b) {
  if (!aligned) {
    a = __ldg(reinterpret_cast<const uint4 *>(src));
    b = __ldg(reinterpret_cast<const uint4 *>(src) + 1);
    return;
  }
  asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
      : "l"(src));
}

// Four int8 b as bf16, exactly.  With u = b + 128 in 0..255, the bf16 0x4300 + u
// is f = 128 + u for u < 128 and 256 + 2 (u - 128) above, so f - 256 is b, or 2 b
// where b > 0; relu(f / 2 - 128) is what is too much.  Three operations of a pair
// go to the fp16 pipe and 1.5 to the integer pipe.
__device__ __forceinline__ uint2 s8x4_to_bf16(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t f[2] = {__byte_perm(u, 0x43434343u, 0x5140), __byte_perm(u, 0x43434343u, 0x5342)};
  uint32_t x[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t d, over;  // constants as bits: 0.5, -128, 256 (a conversion at run time otherwise)
    asm("fma.rn.relu.bf16x2 %0, %1, %2, %3;" : "=r"(over) : "r"(f[i]), "r"(0x3f003f00u), "r"(0xc300c300u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(f[i]), "r"(0x43804380u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(x[i]) : "r"(d), "r"(over));
  }
  return make_uint2(x[0], x[1]);
}

}  // namespace treek

using namespace treek;

// The CTA's items; descriptors are read one item ahead.
struct Items {
  const TreeItem *items;
  TreeItem ahead;
  bool more = true;
  __device__ __forceinline__ explicit Items(const TreeItem *p) : items(p), ahead(p[blockIdx.x]) {}
  __device__ __forceinline__ bool next(TreeItem &im) {
    if (!more) return false;
    im = ahead;
    more = im.next >= 0;
    if (more) ahead = items[im.next];
    return true;
  }
};

// Waits until unit u = 2 step + half is done (or full).  A wait knows its phase
// by parity only, so nobody may ask for a step that is kSteps or more behind the
// last one done, nor ahead of one that is not done.  Step j + 3 is loaded once
// step j is done, and a tile is done only after the softmax has delivered its P:
// while the softmax works on tile j nothing past j + 2 is done (and j + 2 only as
// the next query, whose copy waits for scores alone), and the oldest step it asks
// for is j - 2, the tile before the last query: four behind.  A converter group
// takes every second tile and may ask for step j - 3 when the last it knows done
// is the query at j - 7, while the tile at j - 8 still runs: five ahead.  So six
// barriers a unit are needed, and eight are a mask.  (With four, items of two
// tiles ran past it; tests/test_tree_ring_cpu.py runs the roles in random orders.)
__device__ __forceinline__ bool wait_done(Bars *B, uint32_t u, volatile int *abort, uint32_t *err) {
  return mbar_wait(&B->done[u & 1][(u >> 1) % kSteps], step_phase(u >> 1), abort, err, ERR_TIMEOUT_EMPTY);
}
__device__ __forceinline__ bool wait_full(Bars *B, uint32_t u, volatile int *abort, uint32_t *err) {
  return mbar_wait(&B->full[u & 1][(u >> 1) % kSteps], step_phase(u >> 1), abort, err, ERR_TIMEOUT_FULL);
}

// One CTA per SM, roles by warp:
//   0      TMA producer: queries, ropes, bf16 latents
//   1, 3   tcgen05 issuers, of the scores and of P.V: a commit holds its thread
//          until the MMAs before it have left the queue, so one thread for both
//          leaves the tensor core idle 500 of a tile's 2150 cycles
//   2      loader of the query's rope box
//   4-11   softmax and epilogue.  Scores: warp w has node w % 4 of the group (its
//          16 heads) and the keys 32 ((w - 4) / 4) .. + 31 of a tile; thread l the
//          heads l / 4 and + 8 and eight of the keys (tmem_ld_16x32).  O: thread l
//          has row 32 (w % 2) + l and 128 columns.  With four warps the softmax of
//          a Q8 tile took 2500 cycles and bounded the kernel.
//   12-27  Q8: latents from global memory, as bf16 into the ring
//
// The latent ring runs in steps of two units, half a tile each.  An item is a
// step of query boxes, which the issuer copies to tensor memory (tcgen05.cp),
// then one step a tile.
//
// What bounds it.  One sequence of 131072 rows, 4 nodes: DRAM, 6.8 TB/s while the
// tiles run, 40 us with the merge.  16 of 32768, 64 nodes: the tensor core, 1760
// cycles of a tile's 2050, 1227 us (952 TFLOP/s) under the power cap.  64 of 512 to
// 8192, 8 nodes: 124 us.  Q8 (4 of 32768, 32 nodes: 234 us): a tile takes about 3700
// cycles, for its scores wait until the softmax has read those before, and the
// converters take issue slots and shared memory from both.
template <bool Q8>
__global__ void __launch_bounds__(threads<Q8>(), 1) tree_attend_kernel(const __grid_constant__ TreeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Bars *B = reinterpret_cast<Bars *>(smem + OFF_BAR);
  Scales &scales = *reinterpret_cast<Scales *>(smem + OFF_BAR + sizeof(Bars));
  const uint32_t s_base = smem_u32(smem);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  volatile int *abort = &B->abort;

  // ---- the producer (thread 0): one step a call, false at the end
  TreeItem pim;
  pim.next = blockIdx.x;
  pim.tile1 = 0;
  int pt = 0;
  uint32_t pg = 0, pj = 0;  // tiles and steps issued
  uint32_t step1 = 0, step2 = 0;  // steps of the last tile issued and of the one before
  auto produce = [&]() -> bool {
    // the places of step pj: their last steps must be done
    auto free_unit = [&](int h) -> bool {
      const uint32_t u = 2 * pj + h;
      return u < kUnits || wait_done(B, u - kUnits, abort, p.err);
    };
    if (pt == pim.tile1) {
      if (pim.next < 0) return false;
      pim = p.items[pim.next];
      pt = pim.tile0;
      for (int h = 0; h < 2; ++h) {
        if (!free_unit(h)) return false;
        // two pairs of boxes; a pair's rows alternate, 16 of the even box and 16
        // of the odd one, as their lanes do
        uint64_t *full = &B->full[h][pj % kSteps];
        mbar_arrive_expect_tx(full, kUnit);
        for (int b = 0; b < 2; ++b)
          tma_load_5d(smem + ((2 * pj + h) % kUnits) * kUnit + b * 2 * kBox, &p.tm_q, full, 0, 0, 0, 2 * h + b, pim.node0);
        if (Q8)  // the barrier counts the converter warps
          for (int i = 1; i < kConvertThreads / 32; ++i) mbar_arrive(full);
      }
      ++pj;
      return true;
    }
    const int32_t y = static_cast<int32_t>(pim.row0 + static_cast<long long>(kTreeKeys) * pt);
    for (int h = 0; h < 2 && !Q8; ++h) {
      if (!free_unit(h)) return false;
      uint64_t *full = &B->full[h][pj % kSteps];
      mbar_arrive_expect_tx(full, kUnit + h * kBox);
      tma_load_3d(smem + ((2 * pj + h) % kUnits) * kUnit, &p.tm_lat, full, 0, y, 4 * h);
    }
    if constexpr (Q8) {
      // The rope goes where the second part of the weights of tile pg - 2 lies until
      // its P.V is done, about when the scores of tile pg begin, which need it last:
      // its way from DRAM is taken one tile earlier.
      if (pt + 1 < pim.tile1)
        tma_prefetch_l2_2d(&p.tm_rope, 0, y + kTreeKeys);
      else if (pim.next >= 0)
        tma_prefetch_l2_2d(&p.tm_rope, 0,
                           static_cast<int32_t>(p.items[pim.next].row0 + kTreeKeys * p.items[pim.next].tile0));
      if (pg >= 2 && !wait_done(B, 2 * step2 + 1, abort, p.err)) return false;
      step2 = step1;
      step1 = pj;
      mbar_arrive_expect_tx(&B->r_full[pg & 1], kBox);
      tma_load_2d(smem + OFF_R + (pg & 1) * kBox, &p.tm_rope, &B->r_full[pg & 1], 0, y);
    } else {
      if (pg >= 2 && !mbar_wait(&B->s_full[pg & 1], ((pg >> 1) & 1) ^ 1, abort, p.err, ERR_TIMEOUT_EMPTY)) return false;
      tma_load_2d(smem + OFF_R + (pg & 1) * kBox, &p.tm_rope, &B->full[1][pj % kSteps], kLatent, y);
    }
    ++pt;
    ++pg;
    ++pj;
    return true;
  };

  if (threadIdx.x == 0) {
    for (int h = 0; h < 2; ++h)
      for (uint32_t i = 0; i < kSteps; ++i) {
        mbar_init(&B->full[h][i], Q8 ? kConvertThreads / 32 : 1);
        mbar_init(&B->done[h][i], 1);
      }
    mbar_init(&B->qr_full, 1);
    mbar_init(&B->q_done, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->r_full[i], 1);
      mbar_init(&B->s_full[i], 1);
      mbar_init(&B->s_empty[i], kSoftThreads / 32);
    }
    mbar_init(&B->p_full, kSoftThreads / 32);
    mbar_init(&B->o_empty, kSoftThreads / 32);
    mbar_init(&B->drain[0], 1);
    mbar_init(&B->drain[1], 1);
    B->abort = 0;
    if (s_base & 1023) {  // the swizzle atoms
      B->abort = 1;
      atomicOr(p.err, ERR_BAD_PARAM);
    }
    fence_barrier_init();
    // The first loads go out before the CTA's set-up is done; nothing but the
    // plan is read before the kernel ahead of this one on the stream is complete.
    tma_prefetch_desc(&p.tm_q);
    tma_prefetch_desc(&p.tm_rope);
    if (!Q8) tma_prefetch_desc(&p.tm_lat);
    pdl_wait();
    for (int i = 0; i < 2 && !B->abort; ++i)  // the query and a tile: their places are free
      if (!produce()) break;
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
  pdl_wait();
  pdl_trigger();

  // Q8: 896 threads start with 72 registers each; 72 + 2 x 88 + 4 x 64 = 7 x 72
  if (warp < 4) {
    if (warp == 0 && fit) {
      if (lane == 0) {
        while (produce()) {
        }
        if (*abort) {  // copies in flight land before the CTA exits; no barrier tells of a half-issued step
          const uint64_t from = globaltimer();
          while (globaltimer() - from < 1000000ull) {
          }
        }
      }
    } else if (warp == 1 && fit) {
      if (elect_one()) {
        constexpr uint32_t id_qk = idesc_f16(1, 1, 0, 0, kTreeRows, kTreeKeys);  // both K-major
        const uint32_t k_lo = desc_lo(s_base, 16);
        uint32_t g = 0, j = 0;
        bool ok = true;
        Items items(p.items);
        TreeItem im;
        for (int n = 0; ok && items.next(im); ++n) {
          const int t0 = im.tile0, t1 = im.tile1;
          // ---- the query's boxes to tensor memory, once the scores before have read theirs
          if (n > 0) ok = mbar_wait(&B->q_done, (n - 1) & 1, abort, p.err, ERR_TIMEOUT_MMA);
          if (ok) ok = wait_full(B, 2 * j, abort, p.err) && wait_full(B, 2 * j + 1, abort, p.err);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int c = 0; c < 8; ++c)
              tmem_cp_128x128b(tmem + kColQ + 32 * b + 4 * c,
                               desc_of(k_lo + ((2 * j + (b >> 1)) % kUnits) * kU16 + (b & 1) * 2 * kB16 + c));
          mma_commit(&B->done[0][j % kSteps]);
          mma_commit(&B->done[1][j % kSteps]);
          ++j;
          for (int t = t0; t < t1; ++t, ++j, ++g) {
            // ---- S = Q . K^T
            ok = wait_full(B, 2 * j, abort, p.err);
            // the place of the scores is free: bf16 those of tile g - 2, Q8 of tile g - 1
            const uint32_t before = Q8 ? g - 1 : g - 2;
            if (ok && g >= (Q8 ? 1 : 2))
              ok = mbar_wait(&B->s_empty[before & 1], (before >> 1) & 1, abort, p.err, ERR_TIMEOUT_EMPTY);
            if (ok && t == t0) ok = mbar_wait(&B->qr_full, n & 1, abort, p.err, ERR_TIMEOUT_FULL);
            if (!ok) break;
            tc_fence_after();
            const uint32_t s_lat = tmem + kColS + (Q8 ? 0 : 64 * (g & 1)), s_rope = Q8 ? tmem + kColRope : s_lat;
            // opaque, or the compiler keeps all operand addresses in registers across tiles
            uint32_t tq = tmem + kColQ, kl = k_lo;
            asm volatile("" : "+r"(tq), "+r"(kl));
            bool hi_ok = false;
#pragma unroll
            for (int b = 0; b < 8; ++b) {
              const uint32_t s = (2 * j + (b >> 2)) % kUnits, odd = b & 1 ? kOddLanes : 0;
              if (b == 3) hi_ok = mbar_test(&B->full[1][j % kSteps], step_phase(j));  // MMAs are queued meanwhile
              if (b == 4) {
                if (!hi_ok) ok = wait_full(B, 2 * j + 1, abort, p.err);
                if (!ok) break;
                tc_fence_after();
              }
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_f16_ts(s_lat + odd, tq + 32 * (b >> 1) + 8 * kk + odd,
                           desc_of(kl + s * kU16 + (b & 3) * kB16 + kk * 2), id_qk, b > 1 || kk > 0);
            }
            if (Q8 && ok) {
              ok = mbar_wait(&B->r_full[g & 1], (g >> 1) & 1, abort, p.err, ERR_TIMEOUT_FULL);
              tc_fence_after();
            }
            if (!ok) break;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f16_ss(s_rope, desc_of(kl + OFF_QR / 16 + kk * 2), desc_of(kl + OFF_R / 16 + (g & 1) * kB16 + kk * 2),
                         id_qk, Q8 ? kk > 0 : 1u);
            mma_commit(&B->s_full[g & 1]);
            if (t + 1 == t1) mma_commit(&B->q_done);
          }
        }
        // issued tensor-core work ends before tensor memory is released
        mma_commit(&B->drain[0]);
        drain_wait(&B->drain[0], 0, p.err);
      }
    } else if (warp == 3 && fit) {
      if (elect_one()) {
        constexpr uint32_t id_pv = idesc_f16(1, 1, 0, 1, kTreeRows, 256);  // V rows as they lie: MN-major
        const uint32_t p_lo = desc_lo(s_base + OFF_P, 16), v_lo = desc_lo(s_base, kBox);
        uint32_t g = 0, j = 0;
        bool ok = true;
        Items items(p.items);
        TreeItem im;
        for (int n = 0; ok && items.next(im); ++n) {
          const int t0 = im.tile0, t1 = im.tile1;
          ++j;  // the query
          for (int t = t0; t < t1; ++t, ++j, ++g) {
            // ---- O += P . V
            if (t == t0 && n > 0) ok = mbar_wait(&B->o_empty, (n - 1) & 1, abort, p.err, ERR_TIMEOUT_EMPTY);
            if (ok)
              ok = wait_full(B, 2 * j, abort, p.err) && wait_full(B, 2 * j + 1, abort, p.err) &&
                   mbar_wait(&B->p_full, g & 1, abort, p.err, ERR_TIMEOUT_FULL);
            if (!ok) break;
            tc_fence_after();
            uint32_t pl = p_lo, vl = v_lo, p2 = p_lo + (OFF_R + (g & 1) * kBox - OFF_P) / 16;
            asm volatile("" : "+r"(pl), "+r"(vl), "+r"(p2));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t s = (2 * j + h) % kUnits;
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                const uint64_t v = desc_of(vl + s * kU16 + kk * 128);
                const uint32_t acc = t > t0 || kk > 0;
                if (!Q8)
                  mma_f16_ws_ss(tmem + 128 * h, desc_of(pl + kk * 2), v, id_pv, acc);
                else if (kk & 1)
                  mma_f16_ws_ss_two<1>(tmem + 128 * h, desc_of(pl + kk * 2), desc_of(p2 + kk * 2), v, id_pv, acc);
                else
                  mma_f16_ws_ss_two<0>(tmem + 128 * h, desc_of(pl + kk * 2), desc_of(p2 + kk * 2), v, id_pv, acc);
              }
              mma_commit(&B->done[h][j % kSteps]);
            }
          }
        }
        mma_commit(&B->drain[1]);
        drain_wait(&B->drain[1], 0, p.err);
      }
    } else if (warp == 2 && fit) {
      if (elect_one()) {
        bool ok = true;
        int n = 0;
        Items items(p.items);
        TreeItem im;
        for (; items.next(im); ++n) {
          const int node0 = im.node0;
          if (n > 0) ok = mbar_wait(&B->q_done, (n - 1) & 1, abort, p.err, ERR_TIMEOUT_EMPTY);
          if (!ok) break;
          mbar_arrive_expect_tx(&B->qr_full, kBox);
          tma_load_2d(smem + OFF_QR, &p.tm_qr, &B->qr_full, kLatent, node0 * kHeads);
        }
        if (!ok) drain_wait(&B->qr_full, (n - 1) & 1, p.err);
      }
    }
  } else if (warp < kConvertWarp) {
    if (Q8) asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    if (fit) {
      const int sub = warp & 3, kh = (warp - 4) >> 2;  // node of the group (lane quarter), half of the keys
      const int tid = threadIdx.x - 128;
      const int ra = 16 * sub + (lane >> 2), c2 = 2 * (lane & 3);  // rows ra and ra + 8; keys 8 i + c2, + 1 of the half
      const uint32_t lanes = static_cast<uint32_t>(32 * sub) << 16;
      const int orow = 32 * (sub & 1) + lane;          // O: the lane's row,
      const uint32_t ocol = tmem + 128 * kh + lanes;   // its columns,
      const int odim = 256 * kh + 128 * (sub >> 1);    // and their dims
      uint32_t g = 0, j = 0;
      uint32_t x = 0;  // exchanges so far
      // a negative scale: the scores change their sign as they are read
      const float scale = fabsf(p.scale_log2);
      bool bad = false;
      // the mask word of this warp's node, drafted rows of its sequence only
      auto load_mask = [&](const TreeItem &im) -> uint64_t {
        const uint64_t w = sub < im.nn ? p.mask[im.node0 + sub] : 0;
        return im.tree < 64 ? w & ((uint64_t(1) << im.tree) - 1) : w;
      };
      int it = blockIdx.x;
      uint64_t mask = load_mask(p.items[it]);
      for (;;) {
        ++j;  // its query
        const int tile0 = p.items[it].tile0, tile1 = p.items[it].tile1, len = p.items[it].len;
        const bool real = sub < p.items[it].nn;  // or the rows hold whatever was there
        float m[2] = {-INFINITY, -INFINITY};
        float2 l[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t cleared = 0;  // bit z: some rows of the item's masked tile with t % 2 = z (it has two at most)
        for (int t = tile0; t < tile1; ++t, ++g, ++j) {
          bad |= !mbar_wait(&B->s_full[g & 1], (g >> 1) & 1, abort, p.err, ERR_TIMEOUT_MMA);
          tc_fence_after();
          const uint32_t col = tmem + kColS + (Q8 ? 0 : 64 * (g & 1)) + 32 * kh + lanes;
          float2 ks[4];  // Q8: the keys' row scales
          float2 s[8];  // [8-key block i][row y]: keys 8 i + c2, + 1
          {
            float s0[16], s1[16], sr[Q8 ? 16 : 1];
            tmem_ld_16x32(col, s0);
            tmem_ld_16x32(col + kOddLanes, s1);
            if constexpr (Q8) {
              tmem_ld_16x32(col + (kColRope - kColS), sr);
              bad |= !wait_full(B, 2 * j + 1, abort, p.err);  // the converters' row scales
#pragma unroll
              for (int i = 0; i < 4; ++i)
                ks[i] = *reinterpret_cast<const float2 *>(scales[g % kScaleRing] + 32 * kh + c2 + 8 * i);
            }
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&B->s_empty[g & 1]);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              s[i] = add2(make_float2(s0[2 * i], s0[2 * i + 1]), make_float2(s1[2 * i], s1[2 * i + 1]));
            if constexpr (Q8) {
#pragma unroll
              for (int i = 0; i < 8; ++i) s[i] = fma2(s[i], ks[i >> 1], make_float2(sr[2 * i], sr[2 * i + 1]));
            }
          }
          const bool masked = kTreeKeys * (t + 1) > len;
          uint32_t seen = 0xffu;  // bit 2 i + z: key 8 i + c2 + z
          if (masked) {
            const int d = kTreeKeys * t - len;  // drafted row of the tile's first key
            const uint64_t vis = d >= 0 ? (d < 64 ? mask >> d : 0)
                                        : (d > -64 ? mask << -d | ((uint64_t(1) << -d) - 1) : ~uint64_t(0));
            const uint32_t v = static_cast<uint32_t>(vis >> (32 * kh)) >> c2;
            seen = (v & 3) | (v >> 6 & 12) | (v >> 12 & 48) | (v >> 18 & 192);
            if (!Q8) {
              // A hidden row gets p = 0, but 0 times an infinity or a NaN of the
              // row itself is NaN in the P.V product.  Such a row gives a score
              // that is not finite with every query (a query that is not finite
              // does so with every row, but only its own): clear those rows.  A
              // node that does see one gets its part at the item's end.
              uint32_t nf[2] = {0, 0};
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                nf[i & 1] |= ((__float_as_uint(s[i].x) & 0x7f800000u) == 0x7f800000u) ? 1u << (2 * (i >> 1)) : 0u;
                nf[i & 1] |= ((__float_as_uint(s[i].y) & 0x7f800000u) == 0x7f800000u) ? 2u << (2 * (i >> 1)) : 0u;
              }
              if (named_bar_or(2, kSoftThreads, ((nf[0] | nf[1]) & ~seen) != 0)) {
                uint32_t all = nf[0] & nf[1];
                for (int o = 4; o < 32; o <<= 1) all &= __shfl_xor_sync(0xffffffffu, all, o);
                uint32_t keys = 0;
                for (int i = 0; i < 4; ++i) keys |= (all >> 2 * i & 3) << (8 * i + c2);
                keys = __reduce_or_sync(0xffffffffu, keys);
                if (lane == 0) B->nonfinite[warp - 4] = keys;
                named_bar_sync(2, kSoftThreads);
                uint32_t rows[2] = {~0u, ~0u};
                for (int i = 0; i < 8; ++i) rows[i >> 2] &= B->nonfinite[i];
                const uint32_t box = tid >> 3 & 7;
                uint8_t *v0 = smem + ((2 * j + (box >> 2)) % kUnits) * kUnit + (box & 3) * kBox + (tid & 7) * 16;
                for (int k = tid >> 6; k < kTreeKeys; k += 4)
                  if (rows[k >> 5] >> (k & 31) & 1) *reinterpret_cast<uint4 *>(v0 + k * 128) = make_uint4(0u, 0u, 0u, 0u);
                if (lane == 0)
                  B->cleared[t & 1][sub][kh] = static_cast<uint32_t>(vis >> (32 * kh)) & (kh ? rows[1] : rows[0]);
                cleared |= 1u << (t & 1);
              }
            }
          }
          if (p.scale_log2 < 0.f)
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = make_float2(-s[i].x, -s[i].y);
          if (masked)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (!(seen >> (2 * (i >> 1)) & 1)) s[i].x = -INFINITY;
              if (!(seen >> (2 * (i >> 1)) & 2)) s[i].y = -INFINITY;
            }
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 8; ++i) mx[i & 1] = fmaxf(mx[i & 1], fmaxf(s[i].x, s[i].y));
          // The reference maxima (of the unscaled scores) move only when some row
          // gets its first score or one that exceeds its by 2^8, then for all rows;
          // else nothing is exchanged.
          bool need = false;
#pragma unroll
          for (int y = 0; y < 2; ++y)
            need |= (mx[y] - m[y]) * scale > 8.0f || (m[y] == -INFINITY && mx[y] > -INFINITY);
          need &= real;
          const bool vote = named_bar_or(1, kSoftThreads, need || bad);
          const uint32_t before = 2 * (t > tile0 ? j - 1 : j - 2) + 1;  // the P before is read until its P.V is done
          const bool p_free = g == 0 || mbar_test(&B->done[1][(before >> 1) % kSteps], step_phase(before >> 1));
          if (vote) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 1));
              mx[y] = fmaxf(mx[y], __shfl_xor_sync(0xffffffffu, mx[y], 2));
              if ((lane & 3) == 0) B->red[x & 1][kh][ra + 8 * y] = mx[y];
            }
            if (named_bar_or(1, kSoftThreads, bad)) {
              bad = true;
              break;
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const float mn = fmaxf(m[y], fmaxf(mx[y], B->red[x & 1][kh ^ 1][ra + 8 * y]));
              const float alpha = m[y] == -INFINITY ? 0.f : ex2((m[y] - mn) * scale);
              if (kh == 0 && (lane & 3) == 0) B->alpha[ra + 8 * y] = alpha;
              l[y] = make_float2(l[y].x * alpha, l[y].y * alpha);
              m[y] = mn;
            }
            ++x;
            if (t > tile0) {
              bad |= !wait_done(B, 2 * (j - 1) + 1, abort, p.err);
              named_bar_sync(1, kSoftThreads);
              tc_fence_after();
              const float alpha = B->alpha[orow];
#pragma unroll
              for (int c = 0; c < 128; c += 16) {
                float o[16];
                tmem_ld16(ocol + c, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] *= alpha;
                tmem_st16(ocol + c, o);
              }
              tmem_wait_st();
            }
          }
          float2 ref[2];  // a row that has seen nothing: exp2(-inf) = 0
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float r = m[y] == -INFINITY ? 0.f : -m[y] * scale;
            ref[y] = make_float2(r, r);
          }
          auto clear_hidden = [&] {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (!(seen >> (2 * (i >> 1)) & 1)) s[i].x = 0.f;
              if (!(seen >> (2 * (i >> 1)) & 2)) s[i].y = 0.f;
            }
          };
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 e = fma2(s[i], make_float2(scale, scale), ref[i & 1]);
            s[i] = make_float2(ex2(e.x), ex2(e.y));
          }
          if (masked) clear_hidden();  // with a scale of 0 the -inf became NaN
#pragma unroll
          for (int i = 0; i < 8; ++i) l[i & 1] = add2(l[i & 1], s[i]);
          if (Q8) {  // O accumulates p * scale * int8 row
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = mul2(s[i], ks[i >> 1]);
            if (masked) clear_hidden();  // a hidden row's scale may be anything
          }
          if (!p_free) bad |= !wait_done(B, before, abort, p.err);
          // The weights enter P.V as bf16, the type of the rows they meet; their sums l
          // stay fp32.  A weight is off by 2^-8 at most, 1.6e-3 in the root mean square,
          // like a bf16 output.  bf16 rows: 0.0017 to 0.0019 in all against 64 bits,
          // 0.0017 with the output's rounding alone (the reference weight is 1, exactly).
          // Q8 weights carry the row scale, so that the int8 rows need none, and are all
          // off: 0.0018 to 0.0025, in short sequences up to twice the output's rounding.
          // What the first part leaves goes in as a second one, 16 bits in all: 0.0017;
          // 4 x 32768 rows, 32 nodes 202 -> 234 us, 64 x 512-8192, 4 nodes 78 -> 88 us
          // (the second products without the collector: 255 and 92).
          const uint32_t at = 2 * sub * 1024 + (lane & 7) * 128 + (((4 * kh + (lane >> 3)) ^ (lane & 7)) * 16);
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = pack_bf16(s[2 * i + y].x, s[2 * i + y].y);
            stmatrix_x4(s_base + OFF_P + at + y * 1024, w[0], w[1], w[2], w[3]);
            if constexpr (Q8) {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = pack_bf16(s[2 * i + y].x - __uint_as_float(w[i] << 16),
                                 s[2 * i + y].y - __uint_as_float(w[i] & 0xffff0000u));
              stmatrix_x4(s_base + OFF_R + (g & 1) * kBox + at + y * 1024, w[0], w[1], w[2], w[3]);
            }
          }
          fence_proxy_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&B->p_full);
        }
        if (bad) break;
        // ---- epilogue
        const TreeItem im = p.items[it];
        bad |= !wait_done(B, 2 * (j - 1) + 1, abort, p.err);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float ly = l[y].x + l[y].y;
          ly += __shfl_xor_sync(0xffffffffu, ly, 1);
          ly += __shfl_xor_sync(0xffffffffu, ly, 2);
          if ((lane & 3) == 0) B->red[x & 1][kh][ra + 8 * y] = ly;
        }
        if (named_bar_or(1, kSoftThreads, bad)) {
          bad = true;
          break;
        }
        tc_fence_after();
        if (im.next >= 0) mask = load_mask(p.items[im.next]);
        const float(&sum)[2][kTreeRows] = B->red[x & 1];
        ++x;
        const float lo = sum[0][orow] + sum[1][orow];
        const float inv = lo == 0.f ? 0.f : 1.0f / lo;  // nothing seen: out = 0, lse = -inf
        if (real && kh == 0 && (lane & 3) < 2) {
          const int y = lane & 1, row = ra + 8 * y;
          const float lr = sum[0][row] + sum[1][row];
          const float lse = lr == 0.f ? -INFINITY : ((y ? m[1] : m[0]) * scale + log2f(lr)) * 0.69314718055994531f;
          if (im.slot >= 0)
            p.part_lse[static_cast<size_t>(im.slot) * kTreeRows + row] = lse;
          else if (p.lse)
            p.lse[static_cast<size_t>(im.node0) * kHeads + row] = lse;
        }
        // A partial keeps the threads' own layout, [64 column quads][128 lanes]
        // float4: every store of a warp is 512 contiguous bytes.  (Row by row,
        // 16 bytes of 32 different rows a store, an item's end took 13000 cycles.)
        // A whole result goes row by row to the output: the CTA's last one through
        // the ring, which is empty by then, and by TMA (from registers, 32 bytes
        // of 32 rows a store, it took 6300 cycles); others from registers, while
        // the ring fills for the next item.
        const bool oreal = orow < im.nn * kHeads, staged = im.slot < 0 && im.next < 0;
        float4 *po = reinterpret_cast<float4 *>(p.part_o) +
                     (static_cast<size_t>(max(im.slot, 0)) * 64 + 32 * kh) * 128 + 32 * sub + lane;
        uint16_t *od = p.out + (static_cast<size_t>(im.node0) * kHeads + orow) * kLatent + odim;
        uint8_t *stage = smem + (odim >> 6) * kBox + (orow >> 3) * 1024 + (orow & 7) * 128;
        // Rare, and apart from the loop below.  A cleared row that the node sees scored
        // -inf, with weight 0 (or its weight was NaN, and so is all of o): 0 times its
        // elements is NaN where they are not finite, whatever other nodes of the group
        // see.  A row whose scores are all -inf gives 0, though O may hold 0 * inf; a
        // partial keeps that, for others may have seen more.
        const bool none = oreal && lo == 0.f && im.slot < 0;
        if ((!Q8 && cleared) || __any_sync(0xffffffffu, none)) {
          const int last = im.tile1 - 1;
#pragma unroll 1
          for (int c = 0; c < 128; c += 16) {
            float o[16];
            tmem_ld16(ocol + c, o);
            tmem_wait_ld();
            for (int z = 0; z < 2 && !Q8; ++z) {
              if (!(cleared >> z & 1)) continue;
              const uint16_t *v0 = p.kv + (im.row0 + kTreeKeys * (last - ((last ^ z) & 1))) * kRow + odim + c;
              for (int half = 0; half < 2; ++half)
                for (uint32_t w = B->cleared[z][orow >> 4][half]; w; w &= w - 1) {
                  const uint16_t *v = v0 + (32 * half + __ffs(w) - 1) * kRow;
#pragma unroll
                  for (int i = 0; i < 16; ++i) o[i] = fmaf(0.f, __bfloat162float(__ushort_as_bfloat16(v[i])), o[i]);
                }
            }
            if (none)
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = 0.f;
            __syncwarp();
            tmem_st16(ocol + c, o);
            tmem_wait_st();
          }
        }
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
          float o[16];
          tmem_ld16(ocol + c, o);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= inv;
          if (staged) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
              *reinterpret_cast<uint4 *>(stage + (c >> 6) * kBox + ((((c & 63) >> 3) + i) ^ (orow & 7)) * 16) =
                  make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]), pack_bf16(o[8 * i + 2], o[8 * i + 3]),
                             pack_bf16(o[8 * i + 4], o[8 * i + 5]), pack_bf16(o[8 * i + 6], o[8 * i + 7]));
          } else if (oreal && im.slot >= 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              po[(c / 4 + i) * 128] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          } else if (oreal) {
            store_bf16x16(od + c, p.out_32, o);
          }
          __syncwarp();
        }
        if (staged) {
          fence_proxy_async_smem();
          named_bar_sync(1, kSoftThreads);
          if (warp == 4 && lane < im.nn) {
            for (int b = 0; b < 8; ++b)
              tma_store_2d(&p.tm_out, smem + b * kBox + lane * 2048, 64 * b, (im.node0 + lane) * kHeads);
            tma_store_wait_read();
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B->o_empty);
        if (im.next < 0) break;
        it = im.next;
      }
    }
  } else if (Q8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    // A thread loads 32 latents of a row at a time, four times a tile.  A warp
    // covers 4 rows x 256 dims, eight whole lines: lane bits 3-4 are the box of
    // 64 dims, bits 1-2 the row, bit 0 the half of the box, so that the eight
    // lanes of a store phase fill the eight 16-byte banks of the swizzle.  The
    // conversion is bound by latencies, not by a pipe: with half as many warps (a
    // tile by all of them, the next one in registers) a tile took 3500 cycles.
    const int tid = (threadIdx.x - 32 * kConvertWarp) % kConvertThreads;
    const uint32_t odd = warp >= kConvertWarp + kConvertThreads / 32;
    const int box = lane >> 3, r = 4 * (tid >> 5) + (lane >> 1 & 3), half = lane & 1;
    const uint32_t last = static_cast<uint32_t>(p.rows - 1);  // below 2^31
    const int8_t *lat = p.lat8 + box * 64 + half * 32;
    // the thread's first 16 bytes of row r in place 0; its others are an xor of bits 4-5 away
    const uint32_t to = s_base + box * kBox + (r >> 3) * 1024 + (r & 7) * 128 + (((4 * half) ^ (r & 7)) << 4);
    const bool aligned = (reinterpret_cast<uintptr_t>(p.lat8) & 31) == 0;
    uint32_t j = 0, g = 0;
    bool ok = fit;
    for (int it = blockIdx.x; it >= 0 && ok; it = p.items[it].next) {
      const uint32_t row0 = static_cast<uint32_t>(p.items[it].row0);
      const int t0 = p.items[it].tile0, t1 = p.items[it].tile1;
      ++j;  // the query
      for (int t = t0; t < t1 && ok; ++t, ++j, ++g) {
        if ((g & 1) != odd) continue;
        const uint32_t first = row0 + kTreeKeys * t;
        const float sc = tid < kTreeKeys ? __ldg(p.lscale + min(first + tid, last)) : 0.f;
        uint4 v[8];  // [unit][rows r and r + 32]
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int8_t *src = lat + static_cast<size_t>(min(first + r + 32 * i, last)) * kLatent;
          load_32(src, aligned, v[2 * i], v[2 * i + 1]);
          load_32(src + 256, aligned, v[4 + 2 * i], v[5 + 2 * i]);
        }
        const uint32_t place = to + 2 * (j % (kUnits / 2)) * kUnit;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t u = 2 * j + h;
          if (ok && u >= kUnits) ok = wait_done(B, u - kUnits, abort, p.err);
          if (!ok) break;
          if (h == 1 && tid < kTreeKeys) scales[g % kScaleRing][tid] = sc;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint4 x = v[4 * h + 2 * i + (c >> 1)];
              const uint2 lo = s8x4_to_bf16(c & 1 ? x.z : x.x), hi = s8x4_to_bf16(c & 1 ? x.w : x.y);
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"((place ^ (c << 4)) + h * kUnit + i * 4096),
                           "r"(lo.x), "r"(lo.y), "r"(hi.x), "r"(hi.y)
                           : "memory");
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&B->full[h][j % kSteps]);
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

bool tree_maps(TreeParams &p, const uint16_t *q, const uint16_t *kv, const uint16_t *rope16, uint16_t *out, int nodes,
               int64_t rows) {
  const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B;
  const uint64_t n = nodes, r = rows, row = kRow * 2;
  const uint64_t qd[5] = {64, kHeads, 2, 4, n}, qs[4] = {row, 128, 256, kHeads * row};
  const uint32_t qb[5] = {64, kHeads, 2, 1, kTreeGroup};
  const uint64_t ld[3] = {64, r, 8}, ls[2] = {row, 128};
  const uint32_t lb[3] = {64, kTreeKeys, 4};
  return make_tmap_nd(&p.tm_q, q, dt, 5, qd, qs, qb, sw) &&
         make_tmap_2d(&p.tm_qr, q, dt, kRow, n * kHeads, row, 64, kTreeRows, sw) &&
         make_tmap_2d(&p.tm_out, out, dt, kLatent, n * kHeads, kLatent * 2, 64, kHeads, sw) &&
         (kv ? make_tmap_nd(&p.tm_lat, kv, dt, 3, ld, ls, lb, sw) &&
                   make_tmap_2d(&p.tm_rope, kv, dt, kRow, r, row, 64, kTreeKeys, sw)
             : make_tmap_2d(&p.tm_rope, rope16, dt, kRope, r, kRope * 2, 64, kTreeKeys, sw));
}

cudaError_t launch_tree_attend(const TreeParams &p, bool q8, int grid, cudaStream_t s) {
  static std::atomic<unsigned long long> opted[2];
  const void *fn = q8 ? reinterpret_cast<const void *>(tree_attend_kernel<true>)
                      : reinterpret_cast<const void *>(tree_attend_kernel<false>);
  cudaError_t e = smem_opt_in(fn, q8 ? smem_bytes<true>() : smem_bytes<false>(), opted[q8]);
  if (e != cudaSuccess) return e;
  ProfScope ps(q8 ? "tree_attend_q8" : "tree_attend_bf16", s);
  if (q8) return launch_dependent(tree_attend_kernel<true>, dim3(grid), dim3(threads<true>()), smem_bytes<true>(), s, p);
  return launch_dependent(tree_attend_kernel<false>, dim3(grid), dim3(threads<false>()), smem_bytes<false>(), s, p);
}

// Combines the partials of the split (sequence, group)s:
//     out = sum_q w_q o_q / sum_q w_q,  w_q = exp(lse_q - max lse),
//     lse = max lse + log sum_q w_q.
// Thread (row or lane, z) of block (entry, quad) has four output dims of one
// query row, as the attend's lane left them, and the parts z, z + Z, ...; the Z
// sums are added in order.  Bound by the latency of its two passes over a few
// parts a thread (lse, then outputs); the outputs lie in L2 mostly.
template <int Z, int LANES, int BATCH>
__global__ void __launch_bounds__(LANES * Z) tree_merge_kernel(uint16_t *out, float *lse, const float *part_o,
                                                               const float *part_lse, const TreeMerge *entries) {
  const TreeMerge e = entries[blockIdx.x];
  const int tid = threadIdx.x % LANES, z = threadIdx.x / LANES, quad = blockIdx.y;
  const int at = blockIdx.z * LANES + tid;  // the attend's lane
  const int row = at & 63, half = at >> 6;
  __shared__ float4 acc_z[Z][LANES];
  __shared__ float max_z[Z][LANES], sum_z[Z][LANES];
  pdl_wait();
  pdl_trigger();
  const bool real = row < e.nn * kHeads;
  const float *ls = part_lse + static_cast<size_t>(e.first) * kTreeRows + row;
  const float4 *os = reinterpret_cast<const float4 *>(part_o) + (static_cast<size_t>(e.first) * 64 + quad) * 128 + at;
  // The loads of BATCH parts are on their way at once, the first batch's outputs
  // before its weights are known.
  float w[BATCH];
  float4 v[BATCH];
  auto load_lse = [&](int q0) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      w[i] = real && q0 + Z * i < e.count ? ls[(q0 + Z * i) * kTreeRows] : -INFINITY;
  };
  auto load_out = [&](int q0) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      v[i] = real && q0 + Z * i < e.count ? os[static_cast<size_t>(q0 + Z * i) * 64 * 128] : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float m = -INFINITY;
  for (int q0 = z + Z * BATCH; q0 < e.count; q0 += Z * BATCH) {
    load_lse(q0);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) m = fmaxf(m, w[i]);
  }
  load_lse(z);
  load_out(z);
#pragma unroll
  for (int i = 0; i < BATCH; ++i) m = fmaxf(m, w[i]);
  if (Z > 1) {
    max_z[z][tid] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Z; ++i) m = fmaxf(m, max_z[i][tid]);
  }
  const float ref = m == -INFINITY ? 0.f : m;  // no part has seen a row: all weights are 0
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
  for (int q0 = z;;) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const float wi = __expf(w[i] - ref);
      sum += wi;
      acc.x = fmaf(wi, v[i].x, acc.x);
      acc.y = fmaf(wi, v[i].y, acc.y);
      acc.z = fmaf(wi, v[i].z, acc.z);
      acc.w = fmaf(wi, v[i].w, acc.w);
    }
    q0 += Z * BATCH;
    if (q0 >= e.count) break;
    load_lse(q0);
    load_out(q0);
  }
  if (Z > 1) {
    acc_z[z][tid] = acc;
    sum_z[z][tid] = sum;
    __syncthreads();
    if (z > 0) return;
    for (int i = 1; i < Z; ++i) {
      const float4 v = acc_z[i][tid];
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
      sum += sum_z[i][tid];
    }
  }
  if (!real) return;
  const size_t orow = static_cast<size_t>(e.node0) * kHeads + row;
  if (lse && quad == 0 && half == 0) lse[orow] = sum == 0.f ? -INFINITY : m + logf(sum);
  if (sum == 0.f) acc = make_float4(0.f, 0.f, 0.f, 0.f);  // also where a part holds 0 * inf
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  const int c = 4 * quad;  // the attend lane's column
  *reinterpret_cast<uint2 *>(out + orow * kLatent + (c >> 7) * 256 + half * 128 + (c & 127)) =
      make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

cudaError_t launch_tree_merge(const TreeParams &p, const TreeMerge *entries, int n, int max_count, cudaStream_t s) {
  if (n <= 0) return cudaSuccess;
  ProfScope ps("tree_merge", s);
  auto launch = [&](auto f, int z, int lanes) {
    return launch_dependent(f, dim3(n, 64, 128 / lanes), dim3(lanes * z), 0, s, p.out, p.lse, (const float *)p.part_o,
                            (const float *)p.part_lse, entries);
  };
  // a few parts a thread: more threads share an entry that has many
  if (max_count <= 8) return launch(tree_merge_kernel<1, 128, 8>, 1, 128);
  if (max_count <= 32) return launch(tree_merge_kernel<4, 128, 8>, 4, 128);
  return launch(tree_merge_kernel<16, 32, 10>, 16, 32);
}

}  // namespace kvl
