// pool_move.cu -- rows of latent pools are moved: the accepted rows of a
// drafted tree slide up behind the cache, runs of rows are forked to new
// places, a pool is compacted.  Every row keeps its bits.
//
// A pool is one array of rows (bf16: [rows][R + DR]) or three (Q8: int8
// [rows][R], fp32 [rows], bf16 [rows][DR]); one launch moves the rows of up to
// 64 pools (the layers of a model, whose sequences lie at the same rows).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <vector>

#include "kvl/mla_cuda.h"
#include "prof.cuh"
#include "sm100.cuh"

#define KVL_EXPORT extern "C" __attribute__((visibility("default")))

namespace kvl {

void set_error_text(const char *msg);

constexpr int kMaxPools = 64;
constexpr int kMaxPath = 64;
constexpr int kMaxRowBytes = 36 * 1024;
constexpr int kMoveRows = 32;   // of a move tile
constexpr size_t kMoveSmem = 220 * 1024;  // of the move kernels' blocks on an SM
constexpr size_t kForkSmem = 84 * 1024;   // of a block that moves runs that do not overlap
constexpr int kMaxStages = 16;            // move tiles in a block's shared memory

// The arrays of up to 64 pools: base pointers, bytes of a row, and the widest
// access (16, 8, 4, 2 or 1 bytes) that all rows of all pools are aligned to.
struct PoolArrays {
  uint8_t *base[3][kMaxPools];
  int row_bytes[3];
  int vec[3];
  int arrays;
  int pools;
};

static int fail(const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  set_error_text(buf);
  return -1;
}

// ------------------------------------------------------------------ accept
struct AcceptParams {
  PoolArrays a;
  const int64_t *base;  // [batch]
  const int *path;      // [batch][max_path]
  const int *count;     // [batch]
  int *kept;            // [batch]
  int batch, max_path;
  long long rows;
};

// A sequence's path is usable when it ascends from at least 0 and its rows lie
// in the pool; `hi` is then its last row.
__device__ __forceinline__ bool accept_span(const AcceptParams &p, int b, long long &lo, long long &hi) {
  const int n = p.count[b];
  lo = p.base[b];
  if (n <= 0 || n > p.max_path || lo < 0 || lo >= p.rows) return false;
  hi = lo + p.path[(size_t)b * p.max_path + n - 1];
  return hi >= lo && hi < p.rows;
}

template <typename V>
__device__ __forceinline__ void accept_array(uint8_t *rows, int row_bytes, const int *src, int n) {
  // One thread owns one column of the sequence's rows and walks the path in
  // order.  src[j] >= j and ascends, so a row is read before it is written:
  // writing row j leaves every later source (>= j + 1) alone.
  for (int c = threadIdx.x; c < row_bytes / (int)sizeof(V); c += blockDim.x) {
    V *col = reinterpret_cast<V *>(rows) + c;
    const size_t pitch = row_bytes / sizeof(V);
    for (int j0 = 0; j0 < n; j0 += 8) {
      V v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + i < n) v[i] = col[pitch * src[j0 + i]];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + i < n && src[j0 + i] != j0 + i) col[pitch * (j0 + i)] = v[i];
    }
  }
}

__global__ void __launch_bounds__(128) tree_accept_kernel(const __grid_constant__ AcceptParams p) {
  __shared__ int src[kMaxPath];
  const int b = blockIdx.x, pool = blockIdx.y;
  const int n = p.count[b];
  long long lo = 0, hi = 0;
  bool ok = n == 0 || accept_span(p, b, lo, hi);
  if (ok && n > 0) {
    for (int j = threadIdx.x; j < n; j += blockDim.x) {
      const int s = p.path[(size_t)b * p.max_path + j];
      ok &= s >= j && (j == 0 || s > p.path[(size_t)b * p.max_path + j - 1]);
      src[j] = s;
    }
    // rows that two sequences claim would be written by two blocks
    for (int o = threadIdx.x; o < p.batch; o += blockDim.x) {
      long long l2, h2;
      if (o != b && accept_span(p, o, l2, h2)) ok &= h2 < lo || l2 > hi;
    }
  }
  ok = __syncthreads_and(ok);
  if (threadIdx.x == 0 && pool == 0 && p.kept) p.kept[b] = ok ? n : -1;
  if (!ok || n == 0) return;
  for (int k = 0; k < p.a.arrays; ++k) {
    const int rb = p.a.row_bytes[k];
    uint8_t *rows = p.a.base[k][pool] + lo * rb;
    switch (p.a.vec[k]) {
      case 16: accept_array<uint4>(rows, rb, src, n); break;
      case 8: accept_array<uint2>(rows, rb, src, n); break;
      case 4: accept_array<uint32_t>(rows, rb, src, n); break;
      case 2: accept_array<uint16_t>(rows, rb, src, n); break;
      default: accept_array<uint8_t>(rows, rb, src, n);
    }
  }
}

// ------------------------------------------------------------------ move
// `n` rows go from row `src` to row `dst`.  In a compaction the tiles
// [dep, dep + deps) read rows that this one overwrites.
struct alignas(16) MoveTile {
  int src, dst;
  int dep;
  uint16_t n, deps;
};

struct MoveParams {
  PoolArrays a;
  const MoveTile *tiles;
  int n_tiles;
  int compact;
  int stages;        // ring kernel: tiles in shared memory at once
  uint32_t *ticket;  // compaction: next (pool, tile)
  uint32_t *read;    // compaction: [pools][tiles], 1 once the tile's rows have been read
  uint32_t *err;
};

template <typename V>
__device__ __forceinline__ void copy_bytes(uint8_t *dst, const uint8_t *src, int bytes) {
  for (int i = threadIdx.x; i < bytes / (int)sizeof(V); i += blockDim.x)
    reinterpret_cast<V *>(dst)[i] = reinterpret_cast<const V *>(src)[i];
}

__device__ __forceinline__ void copy_any(int vec, uint8_t *dst, const uint8_t *src, int bytes) {
  switch (vec) {
    case 16: copy_bytes<uint4>(dst, src, bytes); break;
    case 8: copy_bytes<uint2>(dst, src, bytes); break;
    case 4: copy_bytes<uint32_t>(dst, src, bytes); break;
    case 2: copy_bytes<uint16_t>(dst, src, bytes); break;
    default: copy_bytes<uint8_t>(dst, src, bytes);
  }
}

// Waits until flag `d` of a compaction's tiles is set, within the limit.
__device__ __forceinline__ bool wait_read(const uint32_t *flag) {
  const uint64_t t0 = globaltimer();
  for (;;) {
    uint32_t seen;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(flag) : "memory");
    if (seen) return true;
    if (globaltimer() - t0 > KVL_WAIT_LIMIT_NS) return false;
  }
}

__device__ __forceinline__ void set_read(uint32_t *flag) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flag), "r"(1u) : "memory");
}

// A tile's rows go through shared memory.  In a compaction the blocks take the
// tiles in order (a ticket), and a tile is written only once the tiles before
// it whose sources it overwrites have been read.  Reading never waits for
// another block, and a block reads its tiles in the order of their tickets, so
// the lowest tile not yet written always gets through; its block holds it
// already, so no block waits for one that has not started.

// Rows that bulk copies cannot move (not a multiple of 16 bytes, or not aligned
// to 16): one tile at a time through a block's threads.
__global__ void __launch_bounds__(256) pool_move_any_kernel(const __grid_constant__ MoveParams p) {
  extern __shared__ __align__(16) uint8_t buf[];
  __shared__ uint32_t my;
  const uint32_t total = (uint32_t)p.n_tiles * p.a.pools;
  for (uint32_t t = blockIdx.x;; t += gridDim.x) {
    if (p.compact) {
      __syncthreads();
      if (threadIdx.x == 0) my = atomicAdd(p.ticket, 1u);
      __syncthreads();
      t = my;
    }
    if (t >= total) return;
    const int pool = t / p.n_tiles, ti = t % p.n_tiles;
    const MoveTile tile = p.tiles[ti];
    int at = 0;
    for (int k = 0; k < p.a.arrays; ++k) {
      const int bytes = tile.n * p.a.row_bytes[k];
      copy_any(p.a.vec[k], buf + at, p.a.base[k][pool] + (size_t)tile.src * p.a.row_bytes[k], bytes);
      at += (bytes + 15) & ~15;
    }
    __syncthreads();
    if (p.compact) {
      uint32_t *flags = p.read + (size_t)pool * p.n_tiles;
      if (threadIdx.x == 0) {
        __threadfence();
        set_read(flags + ti);
      }
      const bool late = (int)threadIdx.x < tile.deps && !wait_read(flags + tile.dep + threadIdx.x);
      if (__syncthreads_or(late)) {  // leave the tile unwritten rather than lose an unread row
        if (threadIdx.x == 0) atomicOr(p.err, ERR_TIMEOUT_FULL);
        continue;
      }
    }
    at = 0;
    for (int k = 0; k < p.a.arrays; ++k) {
      const int bytes = tile.n * p.a.row_bytes[k];
      copy_any(p.a.vec[k], p.a.base[k][pool] + (size_t)tile.dst * p.a.row_bytes[k], buf + at, bytes);
      at += (bytes + 15) & ~15;
    }
    __syncthreads();
  }
}

// The same with bulk copies, for arrays of 16-byte rows and arrays of one word
// a row (the Q8 row scales): one warp reads tiles into a ring, one writes them,
// and in a compaction one tells that they were read.
// A tile's reading, the flag that tells of it and its writing overlap those of
// the tiles before and after it.  Array k of tile slot q lies at q * tile bytes
// + `kMoveRows` rows of the arrays before it.
//
// Two blocks an SM.  What bounds it is DRAM: 27 bf16 pools whose 4096-row prompt
// goes to four places take 112 us, the same on Q8 61 us, a prompt of 32768 rows
// once 311 us (at the copy rate: 99, 55 and 316); a pool of 64 sequences of up
// to 8192 rows compacted 98 us, 27 Q8 pools of 31 sequences of up to 1000 rows
// 111 us (92 and 80).  With one tile a block in registers' reach, read by its
// threads and then written, the first took 138 us, the compactions 243 and 250.
// The depth: a copy that nothing orders wants about 150 KB on its way in an SM
// (two bf16 tiles a block; five take 121 us, for more is then read and written
// at once), a compaction all it can get (Q8: two tiles a block 270 us, four 131,
// five 111), for a tile waits in the ring until the flags of others have come.
__global__ void __launch_bounds__(96) pool_move_kernel(const __grid_constant__ MoveParams p) {
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages];
  __shared__ struct {
    MoveTile tile;
    uint32_t t;
  } slot[kMaxStages];
  __shared__ volatile int gave_up[2];  // the writing warp still writes what was read when the reading one gave up
  const int lane = threadIdx.x & 31;
  const uint32_t total = (uint32_t)p.n_tiles * p.a.pools;
  const int stages = p.stages;
  int tile_bytes = 0, bulk_row = 0;
  for (int k = 0; k < p.a.arrays; ++k) {
    tile_bytes += kMoveRows * p.a.row_bytes[k];
    if (p.a.vec[k] == 16) bulk_row += p.a.row_bytes[k];
  }
  if (threadIdx.x == 0) {
    gave_up[0] = gave_up[1] = 0;
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 33);  // each lane's words, and the bulk copies
      mbar_init(&empty[i], p.compact ? 2 : 1);
    }
    fence_barrier_init();
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    // Lane 0 has the ticket of the next round, fetched during this one.
    auto take = [&](uint32_t t) -> uint32_t { return !p.compact ? t + gridDim.x : lane == 0 ? atomicAdd(p.ticket, 1u) : 0; };
    uint32_t t = __shfl_sync(0xffffffffu, p.compact ? take(0) : blockIdx.x, 0), next = take(t);
    MoveTile tile = t < total ? p.tiles[t % p.n_tiles] : MoveTile{};
    for (int i = 0;; ++i) {
      const int q = i % stages;
      if (i >= stages && !mbar_wait(&empty[q], (i / stages - 1) & 1, &gave_up[0], p.err, ERR_TIMEOUT_EMPTY)) return;
      if (lane == 0) {
        slot[q].tile = tile;
        slot[q].t = t;
      }
      if (t >= total) {  // tells the writing warp to stop
        if (lane == 0) mbar_arrive(&full[q]);
        mbar_arrive(&full[q]);
        return;
      }
      const int pool = t / p.n_tiles;
      uint8_t *buf = ring + (size_t)q * tile_bytes;
      if (lane == 0) mbar_arrive_expect_tx(&full[q], tile.n * bulk_row);
      for (int k = 0; k < p.a.arrays; ++k) {
        const uint8_t *src = p.a.base[k][pool] + (size_t)tile.src * p.a.row_bytes[k];
        if (p.a.vec[k] == 16) {
          if (lane == 0) bulk_load(buf, src, tile.n * p.a.row_bytes[k], &full[q]);
        } else if (lane < tile.n) {  // one word a row
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(buf) + 4 * lane), "l"(src + 4 * lane)
                       : "memory");
        }
        buf += kMoveRows * p.a.row_bytes[k];
      }
      cp_async_arrive(&full[q]);
      t = __shfl_sync(0xffffffffu, next, 0);
      if (t < total) {
        tile = p.tiles[t % p.n_tiles];
        next = take(t);
      }
    }
  }
  if (threadIdx.x >= 64) {
    // Tells of the tiles read.  Not the writing warp: the flag's release would
    // wait for that warp's own stores first.
    if (lane != 0) return;
    for (int i = 0;; ++i) {
      const int q = i % stages;
      if (!mbar_wait(&full[q], (i / stages) & 1, &gave_up[1], p.err, ERR_TIMEOUT_FULL)) return;
      const uint32_t t = slot[q].t;
      if (t >= total) return;
      set_read(p.read + t);
      mbar_arrive(&empty[q]);
    }
  }
  for (int i = 0;; ++i) {
    const int q = i % stages;
    if (!mbar_wait(&full[q], (i / stages) & 1, &gave_up[1], p.err, ERR_TIMEOUT_FULL)) break;
    const uint32_t t = slot[q].t;
    if (t >= total) break;
    const MoveTile tile = slot[q].tile;
    const int pool = t / p.n_tiles;
    bool late = false;
    if (p.compact) {
      const uint32_t *flags = p.read + (size_t)pool * p.n_tiles + tile.dep;
      late = lane < tile.deps && !wait_read(flags + lane);
      late = __any_sync(0xffffffffu, late);
      if (late && lane == 0) atomicOr(p.err, ERR_TIMEOUT_FULL);
      asm volatile("fence.proxy.async;" ::: "memory");
    }
    uint8_t *buf = ring + (size_t)q * tile_bytes;
    for (int k = 0; k < p.a.arrays && !late; ++k) {  // late: left unwritten rather than lose an unread row
      uint8_t *dst = p.a.base[k][pool] + (size_t)tile.dst * p.a.row_bytes[k];
      if (p.a.vec[k] == 16) {
        if (lane == 0) bulk_store(dst, buf, tile.n * p.a.row_bytes[k]);
      } else if (lane < tile.n) {
        reinterpret_cast<uint32_t *>(dst)[lane] = reinterpret_cast<const uint32_t *>(buf)[lane];
      }
      buf += kMoveRows * p.a.row_bytes[k];
    }
    __syncwarp();
    if (lane == 0) {
      bulk_commit();
      if (i > 0) {
        bulk_wait_read<1>();  // the tile before has left its slot
        mbar_arrive(&empty[(i - 1) % stages]);
      }
    }
  }
  if (lane == 0) bulk_wait<0>();
}

// Fills the arrays of the pools; checks pointers, row sizes and that no two
// pools overlap (their rows would be moved twice).
static int set_pools(PoolArrays &a, void *const *const arrays[3], const long long row_bytes[3],
                     const int elem[3], int n_arrays, int n_pools, int64_t rows) {
  if (n_pools < 1 || n_pools > kMaxPools) return fail("pools: 1 to %d at once, not %d", kMaxPools, n_pools);
  if (rows < 1 || rows >= (1LL << 31)) return fail("pools: %lld rows", (long long)rows);
  std::memset(&a, 0, sizeof a);
  a.arrays = n_arrays;
  a.pools = n_pools;
  struct Range {
    uintptr_t lo, hi;
  } all[3 * kMaxPools];
  int n = 0;
  for (int k = 0; k < n_arrays; ++k) {
    if (!arrays[k]) return fail("pools: null array");
    if (row_bytes[k] < 1 || row_bytes[k] > kMaxRowBytes) return fail("pools: rows of %lld bytes", row_bytes[k]);
    a.row_bytes[k] = (int)row_bytes[k];
    uintptr_t bits = (uintptr_t)row_bytes[k] | 16;
    for (int i = 0; i < n_pools; ++i) {
      const uintptr_t base = reinterpret_cast<uintptr_t>(arrays[k][i]);
      if (!base) return fail("pools: pool %d is null", i);
      if (base % elem[k]) return fail("pools: pool %d is not aligned to its type", i);
      a.base[k][i] = static_cast<uint8_t *>(arrays[k][i]);
      bits |= base;
      all[n++] = {base, base + (uintptr_t)rows * row_bytes[k]};
    }
    a.vec[k] = (int)(bits & (~bits + 1));
  }
  std::sort(all, all + n, [](const Range &x, const Range &y) { return x.lo < y.lo; });
  for (int i = 1; i < n; ++i)
    if (all[i].lo < all[i - 1].hi) return fail("pools: two of the arrays overlap");
  return 0;
}

static int bf16_pools(PoolArrays &a, uint16_t *const *pools, int n_pools, int64_t rows, int R, int DR) {
  if (!pools || R <= 0 || DR <= 0) return fail("pools: invalid arguments");
  void *const *const arrays[3] = {reinterpret_cast<void *const *>(pools), nullptr, nullptr};
  const long long rb[3] = {2LL * ((long long)R + DR), 0, 0};
  const int elem[3] = {2, 1, 1};
  return set_pools(a, arrays, rb, elem, 1, n_pools, rows);
}

static int q8_pools(PoolArrays &a, int8_t *const *lat8, float *const *scale, uint16_t *const *rope, int n_pools,
                    int64_t rows, int R, int DR) {
  if (!lat8 || !scale || !rope || R <= 0 || DR <= 0) return fail("pools: invalid arguments");
  void *const *const arrays[3] = {reinterpret_cast<void *const *>(lat8), reinterpret_cast<void *const *>(scale),
                                  reinterpret_cast<void *const *>(rope)};
  const long long rb[3] = {R, 4, 2LL * DR};
  const int elem[3] = {1, 4, 2};
  return set_pools(a, arrays, rb, elem, 3, n_pools, rows);
}

static int accept(AcceptParams &p, int batch, const int64_t *base, const int *path, const int *count, int max_path,
                  int *kept, int64_t rows, cudaStream_t s) {
  if (batch < 1 || !base || !path || !count || max_path < 1 || max_path > kMaxPath)
    return fail("tree accept: invalid arguments (paths of 1 to %d)", kMaxPath);
  if ((reinterpret_cast<uintptr_t>(base) & 7) ||
      ((reinterpret_cast<uintptr_t>(path) | reinterpret_cast<uintptr_t>(count) | reinterpret_cast<uintptr_t>(kept)) & 3))
    return fail("tree accept: a pointer is not aligned to its type");
  // the blocks of all pools read the inputs while one of them writes `kept`
  auto meets = [&](const void *x, size_t bytes) {
    const uintptr_t k = reinterpret_cast<uintptr_t>(kept), i = reinterpret_cast<uintptr_t>(x);
    return kept && k < i + bytes && i < k + 4 * (size_t)batch;
  };
  if (meets(base, 8 * (size_t)batch) || meets(path, 4 * (size_t)batch * max_path) || meets(count, 4 * (size_t)batch))
    return fail("tree accept: d_kept overlaps an input");
  p.base = base;
  p.path = path;
  p.count = count;
  p.kept = kept;
  p.batch = batch;
  p.max_path = max_path;
  p.rows = rows;
  ProfScope ps("tree_accept", s);
  tree_accept_kernel<<<dim3(batch, p.a.pools), 128, 0, s>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : fail("tree accept launch failed: %s", cudaGetErrorString(e));
}

}  // namespace kvl

using namespace kvl;

struct KvlMlaMovePlan {
  int device = 0;
  bool compact = false;
  long long rows_needed = 0, moved = 0;
  std::vector<MoveTile> tiles;
  void *d_mem = nullptr;  // error word and ticket, read flags, tiles
  size_t off_tiles = 0;
};

KVL_EXPORT int kvl_mla_tree_accept_bf16(uint16_t *const *d_pools, int n_pools, int64_t rows, int kv_lora_rank,
                                        int rope_dim, int batch, const int64_t *d_base, const int *d_path,
                                        const int *d_count, int max_path, int *d_kept, void *stream) {
  AcceptParams p;
  if (bf16_pools(p.a, d_pools, n_pools, rows, kv_lora_rank, rope_dim) != 0) return -1;
  return accept(p, batch, d_base, d_path, d_count, max_path, d_kept, rows, static_cast<cudaStream_t>(stream));
}

KVL_EXPORT int kvl_mla_tree_accept_q8(int8_t *const *d_latent_q8, float *const *d_latent_scale,
                                      uint16_t *const *d_rope_bf16, int n_pools, int64_t rows, int kv_lora_rank,
                                      int rope_dim, int batch, const int64_t *d_base, const int *d_path,
                                      const int *d_count, int max_path, int *d_kept, void *stream) {
  AcceptParams p;
  if (q8_pools(p.a, d_latent_q8, d_latent_scale, d_rope_bf16, n_pools, rows, kv_lora_rank, rope_dim) != 0) return -1;
  return accept(p, batch, d_base, d_path, d_count, max_path, d_kept, rows, static_cast<cudaStream_t>(stream));
}

KVL_EXPORT int kvl_mla_move_plan_create(KvlMlaMovePlan **plan, int runs, const int64_t *src, const int64_t *dst,
                                        const int64_t *count) {
  if (!plan) return fail("move plan: null plan");
  *plan = nullptr;
  if (runs < 1 || !src || !dst || !count) return fail("move plan: invalid arguments");
  struct Run {
    long long s, d, n;
  };
  KvlMlaMovePlan *p = nullptr;
  try {
    std::vector<Run> v;
    for (int i = 0; i < runs; ++i) {
      if (src[i] < 0 || dst[i] < 0 || count[i] < 0 || src[i] >= (1LL << 31) || dst[i] >= (1LL << 31) ||
          count[i] >= (1LL << 31) || src[i] + count[i] >= (1LL << 31) || dst[i] + count[i] >= (1LL << 31))
        return fail("move plan: run %d is out of range", i);
      if (count[i] > 0) v.push_back({src[i], dst[i], count[i]});
    }
    // no row may be written twice
    std::sort(v.begin(), v.end(), [](const Run &x, const Run &y) { return x.d < y.d; });
    for (size_t i = 1; i < v.size(); ++i)
      if (v[i].d < v[i - 1].d + v[i - 1].n) return fail("move plan: two runs write row %lld", v[i].d);
    // runs that stay where they are keep their place in the order of a
    // compaction (their rows may not be written by another run: checked above)
    p = new KvlMlaMovePlan();
    bool ordered = true, down = true;
    for (size_t i = 0; i < v.size(); ++i) {
      p->rows_needed = std::max(p->rows_needed, std::max(v[i].s, v[i].d) + v[i].n);
      down &= v[i].d <= v[i].s;
      ordered &= i == 0 || v[i].s >= v[i - 1].s + v[i - 1].n;
    }
    // does any run write rows that a run reads?
    std::vector<Run> by_src;
    for (const Run &r : v)
      if (r.s != r.d) by_src.push_back(r);
    std::sort(by_src.begin(), by_src.end(), [](const Run &x, const Run &y) { return x.s < y.s; });
    bool overlap = false;
    long long reach = -1;  // one past the last source row of the runs that start at or before the cursor
    size_t k = 0;
    for (const Run &r : v) {
      if (r.s == r.d) continue;
      for (; k < by_src.size() && by_src[k].s < r.d + r.n; ++k) reach = std::max(reach, by_src[k].s + by_src[k].n);
      overlap |= reach > r.d;  // a source that starts before this destination's end reaches into it
    }
    if (overlap && !(ordered && down)) {
      delete p;
      return fail("move plan: a run writes rows that another reads; that needs runs that all move down, in one order");
    }
    p->compact = overlap;
    if (!overlap)  // a source that goes to several places is read from L2 after the first time
      std::sort(v.begin(), v.end(), [](const Run &x, const Run &y) { return x.s != y.s ? x.s < y.s : x.d < y.d; });
    for (const Run &r : v) {
      if (r.s == r.d) continue;
      p->moved += r.n;
      for (long long o = 0; o < r.n; o += kMoveRows)
        p->tiles.push_back({(int)(r.s + o), (int)(r.d + o), 0, (uint16_t)std::min<long long>(kMoveRows, r.n - o), 0});
    }
    if (p->compact) {
      // sources and destinations both ascend: the tiles whose sources a
      // destination overlaps are neighbours
      size_t lo = 0, hi = 0;
      for (size_t i = 0; i < p->tiles.size(); ++i) {
        MoveTile &t = p->tiles[i];
        while (lo < i && p->tiles[lo].src + p->tiles[lo].n <= t.dst) ++lo;
        while (hi < i && p->tiles[hi].src < t.dst + t.n) ++hi;
        t.dep = (int)lo;
        t.deps = (uint16_t)(std::max(lo, hi) - lo);  // at most one a row of the tile
      }
    }
    if (p->tiles.size() > (1u << 24)) {
      delete p;
      return fail("move plan: too many runs");
    }
    int dev = -1;
    const size_t flags = p->compact ? p->tiles.size() * kMaxPools * sizeof(uint32_t) : 0;
    p->off_tiles = (256 + flags + 255) & ~size_t(255);
    const size_t tile_bytes = p->tiles.size() * sizeof(MoveTile);
    if (cudaGetDevice(&dev) != cudaSuccess || cudaMalloc(&p->d_mem, p->off_tiles + tile_bytes + 16) != cudaSuccess ||
        cudaMemset(p->d_mem, 0, p->off_tiles) != cudaSuccess ||
        (tile_bytes && cudaMemcpy(static_cast<uint8_t *>(p->d_mem) + p->off_tiles, p->tiles.data(), tile_bytes,
                                  cudaMemcpyHostToDevice) != cudaSuccess) ||
        cudaStreamSynchronize(cudaStreamLegacy) != cudaSuccess) {  // the plan can be used on any stream afterwards
      cudaGetLastError();
      cudaFree(p->d_mem);
      delete p;
      return fail("move plan: device memory");
    }
    p->device = dev;
  } catch (...) {
    if (p) cudaFree(p->d_mem);
    delete p;
    return fail("move plan: out of host memory");
  }
  *plan = p;
  return 0;
}

KVL_EXPORT void kvl_mla_move_plan_destroy(KvlMlaMovePlan *plan) {
  if (!plan) return;
  cudaFree(plan->d_mem);
  delete plan;
}

KVL_EXPORT int kvl_mla_move_plan_info(const KvlMlaMovePlan *plan, int *compaction, int64_t *moved_rows) {
  if (!plan) return fail("move plan: null plan");
  if (compaction) *compaction = plan->compact;
  if (moved_rows) *moved_rows = plan->moved;
  return 0;
}

static int move_rows(const KvlMlaMovePlan *plan, MoveParams &p, int64_t rows, cudaStream_t s) {
  int dev = -1, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || dev != plan->device)
    return fail("pool move: the plan belongs to device %d, the current device is %d", plan->device, dev);
  if (rows < plan->rows_needed)
    return fail("pool move: a run ends at row %lld, the pools have %lld", plan->rows_needed, (long long)rows);
  if (plan->tiles.empty()) return 0;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  uint8_t *mem = static_cast<uint8_t *>(plan->d_mem);
  p.tiles = reinterpret_cast<const MoveTile *>(mem + plan->off_tiles);
  p.n_tiles = (int)plan->tiles.size();
  p.compact = plan->compact;
  p.err = reinterpret_cast<uint32_t *>(mem);
  p.ticket = p.err + 1;
  p.read = p.err + 64;
  const long long total = (long long)p.n_tiles * p.a.pools;
  if (total >= (1LL << 31)) return fail("pool move: too many rows");
  size_t smem = 0;
  bool bulk = true;
  for (int k = 0; k < p.a.arrays; ++k) {
    smem += ((size_t)kMoveRows * p.a.row_bytes[k] + 15) & ~size_t(15);
    bulk &= p.a.vec[k] == 16 || (p.a.vec[k] == 4 && p.a.row_bytes[k] == 4);
  }
  if (smem > kMoveSmem) return fail("pool move: rows of %zu bytes", smem / kMoveRows);
  const size_t ring = p.compact ? kMoveSmem / 2 : kForkSmem;
  p.stages = (int)std::min<size_t>(kMaxStages, std::max<size_t>(2, ring / smem));
  bulk &= p.stages * smem <= kMoveSmem;
  const int per_sm = bulk ? (p.stages * smem <= kMoveSmem / 2 ? 2 : 1)
                          : std::max(1, std::min(6, (int)(kMoveSmem / smem)));
  if (bulk) smem *= p.stages;
  const auto kernel = bulk ? pool_move_kernel : pool_move_any_kernel;
  cudaError_t e = cudaSuccess;
  if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e == cudaSuccess && p.compact)
    e = cudaMemsetAsync(p.ticket, 0, 252 + (size_t)total * sizeof(uint32_t), s);
  if (e == cudaSuccess) {
    ProfScope ps("pool_move", s);
    kernel<<<(int)std::min<long long>(total, (long long)per_sm * sms), bulk ? (p.compact ? 96 : 64) : 256, smem, s>>>(p);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? 0 : fail("pool move launch failed: %s", cudaGetErrorString(e));
}

KVL_EXPORT int kvl_mla_pool_move_bf16(const KvlMlaMovePlan *plan, uint16_t *const *d_pools, int n_pools, int64_t rows,
                                      int kv_lora_rank, int rope_dim, void *stream) {
  if (!plan) return fail("pool move: null plan");
  MoveParams p;
  if (bf16_pools(p.a, d_pools, n_pools, rows, kv_lora_rank, rope_dim) != 0) return -1;
  return move_rows(plan, p, rows, static_cast<cudaStream_t>(stream));
}

KVL_EXPORT int kvl_mla_pool_move_q8(const KvlMlaMovePlan *plan, int8_t *const *d_latent_q8,
                                    float *const *d_latent_scale, uint16_t *const *d_rope_bf16, int n_pools,
                                    int64_t rows, int kv_lora_rank, int rope_dim, void *stream) {
  if (!plan) return fail("pool move: null plan");
  MoveParams p;
  if (q8_pools(p.a, d_latent_q8, d_latent_scale, d_rope_bf16, n_pools, rows, kv_lora_rank, rope_dim) != 0) return -1;
  return move_rows(plan, p, rows, static_cast<cudaStream_t>(stream));
}

KVL_EXPORT int kvl_mla_move_check(const KvlMlaMovePlan *plan, void *stream) {
  if (!plan) return fail("move check: null plan");
  uint32_t err = 0;
  if (cudaStreamSynchronize(static_cast<cudaStream_t>(stream)) != cudaSuccess ||
      cudaMemcpy(&err, plan->d_mem, 4, cudaMemcpyDeviceToHost) != cudaSuccess)
    return fail("move check: %s", cudaGetErrorString(cudaGetLastError()));
  if (err) {
    cudaMemset(plan->d_mem, 0, 4);
    cudaStreamSynchronize(cudaStreamLegacy);
    return fail("pool move: device-side error 0x%x", err);
  }
  return 0;
}
