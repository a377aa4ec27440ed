// Blocks of a K/V cache: copied, forked with their sequences, compacted, and the free ones listed, on the GPU.
//
// free_list   ref_counts[i] = max(held[i], 0) + how often the tables' entries in use (columns below ceil(len / 256)) name block i;
//             the blocks with none, in order, and how many.  A sequence that has ended frees its blocks by no longer being in
//             the tables.
// fork        row i of the new tables is row parents[i] of the old ones.  Whole blocks are shared; a begun last block goes to
//             its first new row, the others get the next free block and a copy of the begun one's slots.
// compact     of n live blocks those with ids >= n go to the free ids below n, in order; tables follow.
// copy        blocks, or their first slots, in all planes of all tensors of a cache in one launch.
//
// The tables' side is a few trips to memory one after the other: a fork's is worked out by every thread block for itself, so
// that one launch does it all; counts of all blocks lie in the shared memory of one cluster (ids dealt out in ranges), whose
// barriers separate counting, summing and writing.  Copies are bound by memory alone: a (copy, plane) is cut in equal pieces, so
// that few copies of few planes spread over all SMs.  Measured: a fork of 12 sequences to 48 over 28 layers in 8 bits (520 MB read and
// written) 84 us, 6.2 TB/s; two begun blocks of 28 layers 10.7 us, of which start and plan 4; a compaction of 2.2 GB 367, of which counting 6;
// the free list of 256 x 32 entries 6.3.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "copy_ring.cuh"
#include "sm100.cuh"

namespace nvllm {

constexpr int kCopyThreads = 256, kPlanThreads = 1024, kPlanMaxCluster = 8;
constexpr int kPlanMaxBlocks = NVLLM_PAGES_MAX_BLOCKS;
constexpr int kForkMax = NVLLM_FORK_MAX_ROWS;
constexpr int kManyParts = NVLLM_CACHE_MAX_PARTS, kFewParts = 4;
constexpr int64_t kLeastPiece = 4096;  // bytes of a plane's block that are worth a thread block's trip

template <int MOST>
struct Parts {
  nvllm_cache_part part[MOST];
  int n, planes, value_planes;  // planes of all parts, and of those that are not scales
};

// ---- copies: a thread keeps a ring of pieces of shared memory busy, bulk loads kLead pieces ahead of the bulk stores.  Two such
// blocks to an SM with 6 pieces of 16 KB move 6.1-6.2 TB/s (the copy rate is 6.55): one with 8 pieces is as fast on large copies and
// 1-2 us slower on small ones (three blocks of one layer 6.8 us, 4.5 so: room for the next launch beside it), pieces of 8 KB
// 5.5 TB/s, threads with 16-byte loads and stores 5.2-5.4.
constexpr int kPiece = 16384, kStages = 6, kLead = 2;
constexpr int kRingBytes = kPiece * kStages + 128;  // barriers behind the pieces
static_assert(kStages * 8 <= 128, "barriers");

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
template <int N>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

struct RingIo {
  uint32_t ring, bars;
  unsigned char** to;  // of every stage: where its piece goes
  uint32_t* bytes;     // and how much it is
  template <int N>
  __device__ __forceinline__ void read() { bulk_wait_read<N>(); }
  __device__ __forceinline__ void load(int s, unsigned char* dst, const unsigned char* src, uint32_t n) {
    to[s] = dst;
    bytes[s] = n;
    sm100::mbar_expect_tx(bars + 8 * s, n);
    bulk_load(ring + s * kPiece, src, n, bars + 8 * s);
  }
  __device__ __forceinline__ bool wait(int s, uint32_t parity) { return sm100::mbar_wait(bars + 8 * s, parity); }
  __device__ __forceinline__ void store(int s) { bulk_store(to[s], ring + s * kPiece, bytes[s]); }
  __device__ __forceinline__ void finish() { bulk_wait_all(); }
};

// All copies: `of(c, src, dst, slots)` says what copy c is and whether there is anything to do.  A (copy, plane) of values is cut
// in `pieces` equal parts, an item each; items are dealt out to the blocks in turn.  Scales: threads 32 and on.
template <int MOST, class F>
__device__ __forceinline__ void copy_all(const Parts<MOST>& parts, int copies, uint32_t ring, int* status, F&& of) {
  if (copies == 0) return;
  const uint32_t bars = ring + kPiece * kStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) sm100::mbar_init(bars + 8 * i, 1);
    sm100::mbar_fence_init();
    const int64_t pairs = static_cast<int64_t>(copies) * parts.value_planes;
    int64_t largest = 0;
    for (int i = 0; i < parts.n; ++i) largest = max(largest, static_cast<int64_t>(parts.part[i].slot_bytes) * kBlockSize);
    const int64_t wanted = pairs ? (int64_t{8} * gridDim.x + pairs - 1) / pairs : 1, most = (largest + kLeastPiece - 1) / kLeastPiece;
    const int pieces = static_cast<int>(max(int64_t{1}, min(wanted, most)));
    __shared__ unsigned char* s_to[kStages];
    __shared__ uint32_t s_bytes[kStages];
    RingIo io{ring, bars, s_to, s_bytes};
    CopyRing<kStages, kLead, RingIo> moving{io};
    for (int64_t item = blockIdx.x; item < pairs * pieces && moving.ok; item += gridDim.x) {
      const int64_t pair = item / pieces;
      const int c = static_cast<int>(pair / parts.value_planes), k = static_cast<int>(item - pair * pieces);
      int64_t src, dst;
      int slots;
      if (!of(c, src, dst, slots)) continue;
      int plane = static_cast<int>(pair - static_cast<int64_t>(c) * parts.value_planes), i = 0;
      while (parts.part[i].scale_heads > 0 || plane >= static_cast<int>(parts.part[i].planes)) {
        if (parts.part[i].scale_heads == 0) plane -= static_cast<int>(parts.part[i].planes);
        ++i;
      }
      const nvllm_cache_part& part = parts.part[i];
      unsigned char* plane_at = static_cast<unsigned char*>(part.base) + plane * part.plane_stride;
      const int64_t units = static_cast<int64_t>(slots) * part.slot_bytes / 16, each = (units + pieces - 1) / pieces;
      const int64_t end = min((k + 1) * each, units) * 16;
      for (int64_t at = k * each * 16; at < end && moving.ok; at += kPiece)
        moving.piece(plane_at + dst * part.block_stride + at, plane_at + src * part.block_stride + at,
                     static_cast<uint32_t>(min(end - at, static_cast<int64_t>(kPiece))));
    }
    if (!moving.end()) atomicOr(status, NVLLM_STATUS_TIMEOUT);
  } else if (threadIdx.x >= 32) {
    const int scale_planes = parts.planes - parts.value_planes;
    for (int64_t item = blockIdx.x; item < static_cast<int64_t>(copies) * scale_planes; item += gridDim.x) {
      const int c = static_cast<int>(item / scale_planes);
      int64_t src, dst;
      int slots;
      if (!of(c, src, dst, slots)) continue;
      int plane = static_cast<int>(item - static_cast<int64_t>(c) * scale_planes), i = 0;
      while (parts.part[i].scale_heads == 0 || plane >= static_cast<int>(parts.part[i].planes)) {
        if (parts.part[i].scale_heads > 0) plane -= static_cast<int>(parts.part[i].planes);
        ++i;
      }
      const nvllm_cache_part& part = parts.part[i];
      unsigned char* plane_at = static_cast<unsigned char*>(part.base) + plane * part.plane_stride;
      const float* from = reinterpret_cast<const float*>(plane_at + src * part.block_stride);
      float* to = reinterpret_cast<float*>(plane_at + dst * part.block_stride);
      constexpr int groups = kBlockSize / NVLLM_SCALE_GROUP;
      const int held = (slots + NVLLM_SCALE_GROUP - 1) / NVLLM_SCALE_GROUP;
      for (int e = threadIdx.x - 32; e < part.scale_heads * groups; e += blockDim.x - 32)
        if (e % groups < held) to[e] = from[e];
    }
  }
}

struct CopyParams {
  const int32_t *src, *dst, *slots;  // slots NULL: whole blocks
  const int32_t* count;              // nullable: how many of the copies there are
  int copies, num_blocks;
  int* status;
};

template <int MOST>
__global__ void __launch_bounds__(kCopyThreads) copy_blocks_kernel(const __grid_constant__ Parts<MOST> parts, const CopyParams p) {
  extern __shared__ __align__(128) unsigned char s_ring[];
  pdl_prologue();
  const int copies = p.count ? min(*p.count, p.copies) : p.copies;
  copy_all(parts, copies, smem_u32(s_ring), p.status, [&](int c, int64_t& src, int64_t& dst, int& slots) {
    src = p.src[c];
    dst = p.dst[c];
    slots = p.slots ? max(0, min(p.slots[c], kBlockSize)) : kBlockSize;
    if (src < 0 || dst < 0) return false;
    if (src >= p.num_blocks || dst >= p.num_blocks) {
      atomicOr(p.status, NVLLM_STATUS_BAD_BLOCK);
      return false;
    }
    return src != dst;
  });
}

__device__ __forceinline__ int blocks_of(int tokens) { return (tokens + kBlockSize - 1) / kBlockSize; }

// Exclusive prefix sum of `v` over the threads of the block; the total goes to *total.
template <int THREADS>
__device__ __forceinline__ int scan_block(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  int before = incl - v, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  *total = all;
  return before;
}

// ---- fork --------------------------------------------------------------------------------------

struct ForkParams {
  const int32_t* table;
  int64_t stride;
  const int32_t *lens, *parents, *free_blocks;
  int batch, rows, width, n_free, num_blocks;
  int32_t* new_table;
  int64_t new_stride;
  int32_t *new_lens, *taken;
  int* status;
};

template <int MOST>
__global__ void __launch_bounds__(kCopyThreads) fork_kernel(const __grid_constant__ Parts<MOST> parts, const ForkParams p) {
  extern __shared__ __align__(128) unsigned char s_ring[];
  int* s_mem = reinterpret_cast<int*>(s_ring + kRingBytes);
  int* s_first = s_mem;               // of every old sequence: its first new row
  int* s_len = s_first + p.batch;     // and its length
  int* s_fresh = s_len + p.batch;     // of every new row: the block of its own that it gets, -1 none left, -2 none needed
  int4* s_list = reinterpret_cast<int4*>(s_mem + ((2 * p.batch + p.rows + 3) & ~3));  // copies: from, to, slots
  __shared__ int s_warp[kCopyThreads / 32];
  const int tid = threadIdx.x;
  pdl_prologue();
  const int most = p.width * kBlockSize;
  bool bad = false;
  int parent = tid < p.rows ? p.parents[tid] : -1;  // in flight with the lengths
  for (int b = tid; b < p.batch; b += kCopyThreads) {
    const int n = p.lens[b], len = max(0, min(n, most));
    s_first[b] = 0x7fffffff;
    s_len[b] = len;
    if (n != len) s_len[b] = len | static_cast<int>(0x80000000u);  // marked: an error if a row goes on from it
  }
  __syncthreads();
  for (int i = tid; i < p.rows; i += kCopyThreads) {
    const int b = i == tid ? parent : p.parents[i];
    if (b >= 0 && b < p.batch) {
      atomicMin(&s_first[b], i);
      bad |= s_len[b] < 0;
    } else {
      bad |= b >= p.batch;
    }
  }
  __syncthreads();
  auto length = [&](int b) { return b < 0 || b >= p.batch ? 0 : s_len[b] & 0x7fffffff; };
  const int per = (p.rows + kCopyThreads - 1) / kCopyThreads, lo = min(tid * per, p.rows), hi = min(lo + per, p.rows);
  int sum = 0;
  for (int i = lo; i < hi; ++i) {
    const int b = p.parents[i], n = length(b);
    const bool copied = n % kBlockSize && s_first[b] < i;
    s_fresh[i] = copied;
    sum += copied;
  }
  int total;
  int k = scan_block<kCopyThreads>(sum, s_warp, &total);
  for (int i = lo; i < hi; ++i) {
    if (!s_fresh[i]) {
      s_fresh[i] = -2;
      continue;
    }
    const int b = p.parents[i], n = length(b), to = k < p.n_free ? p.free_blocks[k] : -1;
    s_fresh[i] = to;
    s_list[k++] = make_int4(p.table[b * p.stride + blocks_of(n) - 1], to, n % kBlockSize, 0);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (bad) atomicOr(p.status, NVLLM_STATUS_BAD_BLOCK);
    for (int i = tid - 32; i >= 0 && i < p.rows; i += kCopyThreads - 32) p.new_lens[i] = length(p.parents[i]);
    if (tid == 32) *p.taken = total;
  }
  // the tables, while the first thread copies
  constexpr int writers = kCopyThreads - 32;
  for (unsigned e = blockIdx.x * writers + tid - 32; tid >= 32 && e < static_cast<unsigned>(p.rows) * p.width; e += gridDim.x * writers) {
    const int i = static_cast<int>(e / p.width), col = static_cast<int>(e - i * p.width);
    const int b = p.parents[i], need = blocks_of(length(b)), fresh = s_fresh[i];
    int id = -1;
    if (col < need) id = col == need - 1 && fresh != -2 ? fresh : p.table[b * p.stride + col];
    p.new_table[i * p.new_stride + col] = id;
  }
  copy_all(parts, total, smem_u32(s_ring), p.status, [&](int c, int64_t& src, int64_t& dst, int& slots) {
    const int4 x = s_list[c];
    src = x.x;
    dst = x.y;
    slots = x.z;
    if (src < 0 || dst < 0) return false;
    if (src >= p.num_blocks || dst >= p.num_blocks) {
      atomicOr(p.status, NVLLM_STATUS_BAD_BLOCK);
      return false;
    }
    return src != dst;
  });
}

// ---- counts of all blocks ------------------------------------------------------------------------

struct PlanParams {
  const int32_t* table;
  int64_t stride;
  const int32_t *lens, *held;  // held nullable
  int batch, width, num_blocks;
  // free_list
  int32_t *ref_counts, *free_blocks, *num_free;
  // compact
  int32_t *holes, *movers, *moves;  // scratch: free ids below num_live, live ids from it on, how many
  int32_t* new_table;
  int64_t new_stride;
  int32_t *moved_to, *num_live;
  int* status;
};

template <bool COMPACT, bool SEVERAL>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanParams p) {
  namespace cg = cooperative_groups;
  extern __shared__ int s_count[];  // of the ids [first, first + mine)
  __shared__ int s_warp[kPlanThreads / 32], s_free[kPlanMaxCluster], s_holes;
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = SEVERAL ? static_cast<int>(cluster.num_blocks()) : 1, crank = SEVERAL ? static_cast<int>(cluster.block_rank()) : 0;
  const int tid = threadIdx.x;
  const int share = (p.num_blocks + csize - 1) / csize, first = crank * share, mine = max(0, min(share, p.num_blocks - first));
  const int me = crank * kPlanThreads + tid, all = csize * kPlanThreads;
  auto sync = [&]() {
    if constexpr (SEVERAL) cluster.sync();
    else __syncthreads();
  };
  auto at_rank = [&](int* mem, int r) {
    if constexpr (SEVERAL) return cluster.map_shared_rank(mem, r);
    else return mem;
  };
  auto count_of = [&](int id) {
    const int owner = SEVERAL ? id / share : 0;
    return at_rank(s_count, owner) + (id - owner * share);
  };
  pdl_prologue();

  // The entries in use, a few of a thread in flight at a time: f(entry, id), a negative id where there is none.
  const int most = p.width * kBlockSize, entries = p.batch * p.width;
  constexpr int E = 8;
  bool bad = false;
  int id[E], len[E];
  auto load = [&](int from) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const unsigned e = from + k * all;
      if (e < static_cast<unsigned>(entries)) {
        const int b = e / static_cast<unsigned>(p.width);
        len[k] = p.lens[b];
        id[k] = p.table[b * p.stride + (e - b * p.width)];
      }
    }
  };
  auto each = [&](int from, auto&& f) {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const unsigned e = from + k * all;
      if (e >= static_cast<unsigned>(entries)) continue;
      const int col = e % static_cast<unsigned>(p.width), n = len[k];
      bad |= n < 0 || n > most;
      const bool used = col < blocks_of(max(0, min(n, most)));
      bad |= used && id[k] >= p.num_blocks;
      f(e, used && id[k] < p.num_blocks ? id[k] : -1);
    }
  };
  load(me);
  for (int i = tid; i < mine; i += kPlanThreads) s_count[i] = p.held ? max(p.held[first + i], 0) : 0;
  sync();
  for (int from = me;;) {
    each(from, [&](int, int i) {
      if (i >= 0) atomicAdd(count_of(i), 1);
    });
    if (entries - from <= E * all) break;
    from += E * all;
    load(from);
  }
  if (bad) atomicOr(p.status, NVLLM_STATUS_BAD_BLOCK);
  sync();

  // free ids before those of a thread, which has a run of them (odd: no two of a warp in one bank)
  const int run = ((mine + kPlanThreads - 1) / kPlanThreads) | 1, lo = min(tid * run, mine), hi = min(lo + run, mine);
  int sum = 0, total;
  for (int i = lo; i < hi; ++i) sum += s_count[i] == 0;
  int before = scan_block<kPlanThreads>(sum, s_warp, &total);
  int free_all = total;
  if constexpr (SEVERAL) {
    if (tid < csize) cluster.map_shared_rank(s_free, tid)[crank] = total;
    cluster.sync();
    free_all = 0;
    for (int r = 0; r < csize; ++r) {
      if (r < crank) before += s_free[r];
      free_all += s_free[r];
    }
  }
  if constexpr (!COMPACT) {
    for (int i = lo; i < hi; ++i)
      if (s_count[i] == 0) p.free_blocks[before++] = first + i;
    for (int i = tid; i < mine; i += kPlanThreads) p.ref_counts[first + i] = s_count[i];
    for (int i = free_all + me; i < p.num_blocks; i += all) p.free_blocks[i] = -1;
    if (me == 0) *p.num_free = free_all;
  } else {
    const int live = p.num_blocks - free_all;
    int f = before;
    for (int i = lo; i < hi; ++i) {  // free ids before id `live`: the holes, as many as blocks move
      if (first + i == live)
        for (int r = 0; r < csize; ++r) at_rank(&s_holes, r)[0] = f;
      f += s_count[i] == 0;
    }
    if (live == p.num_blocks && tid == 0) s_holes = 0;
    sync();
    const int holes = s_holes;
    f = before;
    for (int i = lo; i < hi; ++i) {
      const int b = first + i;
      if (s_count[i] == 0) {
        if (b < live) p.holes[f] = b;
        ++f;
      } else if (b >= live) {
        p.movers[b - f - (live - holes)] = b;
      }
    }
    sync();
    f = before;
    for (int i = lo; i < hi; ++i) {
      const int b = first + i;
      int to = b;
      if (s_count[i] == 0) {
        ++f;
        to = -1;
      } else if (b >= live) {
        to = __ldcg(p.holes + (b - f - (live - holes)));
      }
      s_count[i] = to;
    }
    sync();
    for (int i = tid; i < mine; i += kPlanThreads) p.moved_to[first + i] = s_count[i];
    for (int from = me; from < entries; from += E * all) {
      if (entries > E * all) load(from);  // else the thread still has its entries
      each(from, [&](int e, int i) {
        const int b = e / p.width;
        p.new_table[b * p.new_stride + (e - b * p.width)] = i >= 0 ? *count_of(i) : -1;
      });
    }
    if (me == 0) {
      *p.num_live = live;
      *p.moves = holes;
    }
    if constexpr (SEVERAL) cluster.sync();  // the others read this block's shared memory
  }
}

// ---- host ----------------------------------------------------------------------------------------

static int check_parts(const char* what, const nvllm_cache_part* part, int n, int64_t num_blocks) {
  if (n <= 0 || n > kManyParts) return fail(NVLLM_E_GEOMETRY, "%s: %d tensors of a cache, outside 1 to %d", what, n, kManyParts);
  if (num_blocks <= 0 || num_blocks > 0x7fffffff / kBlockSize) return fail(NVLLM_E_GEOMETRY, "%s: num_blocks=%lld invalid", what, (long long)num_blocks);
  if (!part) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", what);
  int64_t planes = 0;
  for (int i = 0; i < n; ++i) {
    const nvllm_cache_part& c = part[i];
    if (!c.base) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", what);
    const bool scales = c.scale_heads > 0;
    const int64_t bytes = scales ? static_cast<int64_t>(c.scale_heads) * (kBlockSize / NVLLM_SCALE_GROUP) * 4 : static_cast<int64_t>(c.slot_bytes) * kBlockSize;
    if (c.planes <= 0 || c.scale_heads < 0 || c.slot_bytes < 0 || bytes <= 0 || (scales && c.slot_bytes) || c.block_stride < bytes || (c.planes > 1 && c.plane_stride < bytes))
      return fail(NVLLM_E_GEOMETRY, "%s: tensor %d of the cache has a shape or strides that its blocks do not fit", what, i);
    if (!aligned16(c.base) || c.block_stride % 16 || c.plane_stride % 16 || c.slot_bytes % 16)
      return fail(NVLLM_E_ALIGN, "%s: tensor %d of the cache, its strides and a slot's bytes must be 16-byte aligned", what, i);
    planes += c.planes;
  }
  if (planes > 0xffff) return fail(NVLLM_E_GEOMETRY, "%s: %lld planes are too many", what, (long long)planes);
  return NVLLM_OK;
}

template <int MOST>
static Parts<MOST> gather(const nvllm_cache_part* part, int n) {
  Parts<MOST> all{};
  std::copy(part, part + n, all.part);
  all.n = n;
  for (int i = 0; i < n; ++i) {
    all.planes += static_cast<int>(part[i].planes);
    if (part[i].scale_heads == 0) all.value_planes += static_cast<int>(part[i].planes);
  }
  return all;
}

static int launch_copies(const char* what, const nvllm_cache_part* part, int n, const CopyParams& p, cudaStream_t stream) {
  static bool ready[2][64] = {};
  const int many = n > kFewParts;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[many][dev]) {
    const cudaError_t e = many ? cudaFuncSetAttribute(copy_blocks_kernel<kManyParts>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes)
                               : cudaFuncSetAttribute(copy_blocks_kernel<kFewParts>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
    if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "%s: cannot reserve shared memory: %s", what, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[many][dev] = true;
  }
  const dim3 grid(static_cast<unsigned>(2 * num_sms()));
  if (!many) return launch_kernel(what, copy_blocks_kernel<kFewParts>, grid, dim3(kCopyThreads), kRingBytes, stream, gather<kFewParts>(part, n), p);
  return launch_kernel(what, copy_blocks_kernel<kManyParts>, grid, dim3(kCopyThreads), kRingBytes, stream, gather<kManyParts>(part, n), p);
}

static int check_tables(const char* what, const int32_t* table, int64_t stride, int32_t width, const int32_t* lens, int32_t batch) {
  if (batch < 0 || width <= 0 || stride < width || static_cast<int64_t>(width) * kBlockSize > 0x7fffffff ||
      static_cast<int64_t>(batch) * width > (1 << 28))
    return fail(NVLLM_E_GEOMETRY, "%s: batch=%d max_blocks=%d invalid, beyond the row stride or too many entries", what, batch, width);
  if (batch > 0 && (!table || !lens)) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", what);
  return NVLLM_OK;
}

template <bool COMPACT>
static int launch_plan(const char* what, const PlanParams& p, cudaStream_t stream) {
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  constexpr int most = (kPlanMaxBlocks + kPlanMaxCluster - 1) / kPlanMaxCluster * 4;
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    cudaError_t e = cudaFuncSetAttribute(plan_kernel<COMPACT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(plan_kernel<COMPACT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "%s: cannot reserve shared memory: %s", what, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  // One block up to four entries and blocks to a thread (64 x 16 entries 3.9 us, 256 x 16 entries of 2000 blocks 5.5, a cluster 6.1),
  // then a cluster of eight (256 x 32 of 4200 6.4 us, two blocks 7.5, one 8.8; 512 x 32 of 8000 7.7, two 12).
  const int64_t items = std::max<int64_t>(p.num_blocks, static_cast<int64_t>(p.batch) * p.width);
  const int csize = items <= 4 * kPlanThreads ? 1 : kPlanMaxCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(csize);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>((p.num_blocks + csize - 1) / csize) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = csize;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = csize > 1 ? 2 : 1;
  const cudaError_t e = csize > 1 ? cudaLaunchKernelEx(&cfg, plan_kernel<COMPACT, true>, p) : cudaLaunchKernelEx(&cfg, plan_kernel<COMPACT, false>, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(NVLLM_E_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  }
  count_launch();
  return NVLLM_OK;
}

}  // namespace nvllm

extern "C" int nvllm_copy_blocks(const nvllm_cache_part* parts, int32_t num_parts, int64_t num_blocks, const int32_t* src_blocks,
                                 const int32_t* dst_blocks, const int32_t* num_slots, int64_t num_copies, void* stream) {
  using namespace nvllm;
  if (num_copies < 0 || num_copies > 0x7fffffff) return fail(NVLLM_E_GEOMETRY, "copy_blocks: num_copies=%lld invalid", (long long)num_copies);
  if (const int e = check_parts("copy_blocks", parts, num_parts, num_blocks)) return e;
  if (num_copies == 0) return NVLLM_OK;
  if (!src_blocks || !dst_blocks) return fail(NVLLM_E_NULL, "copy_blocks: NULL pointer argument");
  CopyParams p{src_blocks, dst_blocks, num_slots, nullptr, static_cast<int>(num_copies), static_cast<int>(num_blocks), status_word()};
  if (!p.status || num_sms() <= 0) return fail(NVLLM_E_NO_DEVICE, "copy_blocks: no CUDA device is usable");
  return launch_copies("copy_blocks", parts, num_parts, p, static_cast<cudaStream_t>(stream));
}

extern "C" int nvllm_fork_sequences(const nvllm_cache_part* parts, int32_t num_parts, int64_t num_blocks, const int32_t* block_tables,
                                    int64_t bt_row_stride, int32_t max_blocks, const int32_t* seq_lens, int32_t batch,
                                    const int32_t* parents, int32_t num_rows, const int32_t* free_blocks, int32_t num_free,
                                    int32_t* new_tables, int64_t new_row_stride, int32_t* new_lens, int32_t* blocks_taken, void* stream) {
  using namespace nvllm;
  if (const int e = check_parts("fork_sequences", parts, num_parts, num_blocks)) return e;
  if (const int e = check_tables("fork_sequences", block_tables, bt_row_stride, max_blocks, seq_lens, batch)) return e;
  if (static_cast<int64_t>(num_rows) * max_blocks > (1 << 28)) return fail(NVLLM_E_GEOMETRY, "fork_sequences: %d rows of %d blocks are too many", num_rows, max_blocks);
  if (batch > kForkMax || num_rows <= 0 || num_rows > kForkMax || num_free < 0 || new_row_stride < max_blocks)
    return fail(NVLLM_E_GEOMETRY, "fork_sequences: %d rows from %d outside 1 to %d, num_free=%d, or a short row stride", num_rows, batch, kForkMax, num_free);
  if (!parents || !new_tables || !new_lens || !blocks_taken || (num_free > 0 && !free_blocks))
    return fail(NVLLM_E_NULL, "fork_sequences: NULL pointer argument");
  ForkParams p{block_tables, bt_row_stride, seq_lens, parents, free_blocks, batch, num_rows, max_blocks, num_free, static_cast<int>(num_blocks),
               new_tables, new_row_stride, new_lens, blocks_taken, status_word()};
  if (!p.status || num_sms() <= 0) return fail(NVLLM_E_NO_DEVICE, "fork_sequences: no CUDA device is usable");
  static bool ready[2][64] = {};
  const int many = num_parts > kFewParts;
  int dev = 0;
  cudaGetDevice(&dev);
  auto bytes = [](int64_t old, int64_t rows) { return static_cast<size_t>(kRingBytes + ((2 * old + rows + 3) & ~3ll) * 4 + rows * 16); };
  if (dev < 0 || dev >= 64 || !ready[many][dev]) {
    const int most = static_cast<int>(bytes(kForkMax, kForkMax));
    const cudaError_t e = many ? cudaFuncSetAttribute(fork_kernel<kManyParts>, cudaFuncAttributeMaxDynamicSharedMemorySize, most)
                               : cudaFuncSetAttribute(fork_kernel<kFewParts>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "fork_sequences: cannot reserve shared memory: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[many][dev] = true;
  }
  const dim3 grid(static_cast<unsigned>(2 * num_sms()));
  const size_t smem = bytes(batch, num_rows);
  if (!many)
    return launch_kernel("fork_sequences", fork_kernel<kFewParts>, grid, dim3(kCopyThreads), smem, static_cast<cudaStream_t>(stream),
                         gather<kFewParts>(parts, num_parts), p);
  return launch_kernel("fork_sequences", fork_kernel<kManyParts>, grid, dim3(kCopyThreads), smem, static_cast<cudaStream_t>(stream),
                       gather<kManyParts>(parts, num_parts), p);
}

extern "C" int nvllm_free_list(const int32_t* block_tables, int64_t bt_row_stride, int32_t max_blocks, const int32_t* seq_lens,
                               int32_t batch, const int32_t* held, int64_t num_blocks, int32_t* ref_counts, int32_t* free_blocks,
                               int32_t* num_free, void* stream) {
  using namespace nvllm;
  if (const int e = check_tables("free_list", block_tables, bt_row_stride, max_blocks, seq_lens, batch)) return e;
  if (num_blocks <= 0 || num_blocks > kPlanMaxBlocks) return fail(NVLLM_E_GEOMETRY, "free_list: num_blocks=%lld outside 1 to %d", (long long)num_blocks, kPlanMaxBlocks);
  if (!ref_counts || !free_blocks || !num_free) return fail(NVLLM_E_NULL, "free_list: NULL pointer argument");
  PlanParams p{};
  p.status = status_word();
  if (!p.status) return fail(NVLLM_E_NO_DEVICE, "free_list: no CUDA device is usable");
  p.table = block_tables;
  p.stride = bt_row_stride;
  p.lens = seq_lens;
  p.held = held;
  p.batch = batch;
  p.width = max_blocks;
  p.num_blocks = static_cast<int>(num_blocks);
  p.ref_counts = ref_counts;
  p.free_blocks = free_blocks;
  p.num_free = num_free;
  return launch_plan<false>("free_list", p, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t nvllm_compact_workspace_bytes(int64_t num_blocks) {
  using namespace nvllm;
  if (num_blocks <= 0 || num_blocks > kPlanMaxBlocks)
    return fail(NVLLM_E_GEOMETRY, "compact_blocks: num_blocks=%lld outside 1 to %d", (long long)num_blocks, kPlanMaxBlocks);
  return (num_blocks / 2 * 2 + 4) * 4;
}

extern "C" int nvllm_compact_blocks(const nvllm_cache_part* parts, int32_t num_parts, int64_t num_blocks, const int32_t* block_tables,
                                    int64_t bt_row_stride, int32_t max_blocks, const int32_t* seq_lens, int32_t batch, const int32_t* held,
                                    int32_t* new_tables, int64_t new_row_stride, int32_t* moved_to, int32_t* num_live, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  using namespace nvllm;
  if (const int e = check_parts("compact_blocks", parts, num_parts, num_blocks)) return e;
  if (const int e = check_tables("compact_blocks", block_tables, bt_row_stride, max_blocks, seq_lens, batch)) return e;
  if (new_row_stride < max_blocks) return fail(NVLLM_E_GEOMETRY, "compact_blocks: a row stride is smaller than max_blocks");
  const int64_t need = nvllm_compact_workspace_bytes(num_blocks);
  if (need < 0) return static_cast<int>(need);
  if ((batch > 0 && !new_tables) || !moved_to || !num_live) return fail(NVLLM_E_NULL, "compact_blocks: NULL pointer argument");
  if (!workspace || workspace_bytes < need) return fail(NVLLM_E_WORKSPACE, "compact_blocks: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
  PlanParams p{};
  p.status = status_word();
  if (!p.status || num_sms() <= 0) return fail(NVLLM_E_NO_DEVICE, "compact_blocks: no CUDA device is usable");
  p.table = block_tables;
  p.stride = bt_row_stride;
  p.lens = seq_lens;
  p.held = held;
  p.batch = batch;
  p.width = max_blocks;
  p.num_blocks = static_cast<int>(num_blocks);
  const int half = static_cast<int>(num_blocks / 2);  // no more blocks move than there are holes
  p.moves = static_cast<int32_t*>(workspace);
  p.holes = p.moves + 4;
  p.movers = p.holes + half;
  p.new_table = new_tables;
  p.new_stride = new_row_stride;
  p.moved_to = moved_to;
  p.num_live = num_live;
  if (const int e = launch_plan<true>("compact_blocks", p, static_cast<cudaStream_t>(stream))) return e;
  if (half == 0) return NVLLM_OK;
  const CopyParams c{p.movers, p.holes, nullptr, p.moves, half, static_cast<int>(num_blocks), p.status};
  return launch_copies("compact_blocks", parts, num_parts, c, static_cast<cudaStream_t>(stream));
}
