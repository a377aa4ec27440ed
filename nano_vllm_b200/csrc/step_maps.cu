// step_maps: what tells a step's launches where its rows lie, from the requests' lengths, on the GPU.
//
// Sequence b has cached_lens[b] tokens in the cache and seq_lens[b] with this step.  With held = ceil(cached / 256), need =
// ceil(seq / 256) and first[b] the sum of max(need - held, 0) over the sequences before it:
//   block_tables[b][held .. need) = free_blocks[first[b] ...];  entries from need on: -1;  entries below held stay
//   cu_seqlens_q, cu_seqlens_k: prefix sums of max(seq - cached, 0), cut to the rows there are, and of seq
//   packed token t of b: position cached + t, slot = table[position / 256] * 256 + position % 256
//   rows behind the last token: slot -1 (stored nowhere), position 0
//
// Every thread block sums the lengths itself (two words a sequence, a scan in shared memory) and then fills its share of the
// tables and rows, so one launch does it without any block waiting for another.  A token finds its sequence by bisection of
// the sums; a fresh block's id is read from the free list and not from the table that another block fills.
//
// Bound by trips one after the other (lengths, sums, entries): 2.9 us in a chain of launches for a decode step of 256 sequences
// with tables 16 wide, 4.1 for 512 prompts; three arrays of sums instead of one of 16 bytes a sequence, lengths read twice
// and 64-bit indexes were 4.3 for the former.
#include <algorithm>

#include "common.cuh"

namespace nvllm {

constexpr int kMapsThreads = 256;
constexpr int kMapsMaxBatch = 4096;  // 16 bytes a sequence in shared memory

struct StepMapsParams {
  const int32_t* seq_lens;
  const int32_t* cached_lens;
  int batch;
  int32_t* block_tables;
  int64_t bt_stride;
  int width;
  const int32_t* free_blocks;
  int n_free;
  int32_t* cu_q;
  int32_t* cu_k;
  int32_t* slots;
  int64_t* positions;
  int rows;
  int32_t* taken;
  int* status;
};

__global__ void __launch_bounds__(kMapsThreads) step_maps_kernel(const StepMapsParams p) {
  extern __shared__ int4 s_seq[];  // of every sequence: first packed token, first fresh block, cached tokens, all tokens; then the sums
  __shared__ int s_warp[3][kMapsThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int most = p.width * kBlockSize;
  pdl_wait();
  pdl_trigger();
  auto blocks = [](int tokens) { return (tokens + kBlockSize - 1) / kBlockSize; };

  // per thread a run of sequences; their sums, a scan over the threads, then the run again
  const int per = (p.batch + kMapsThreads - 1) / kMapsThreads;
  const int lo = min(tid * per, p.batch), hi = min(lo + per, p.batch);
  int sum[3] = {0, 0, 0};  // new tokens, fresh blocks, all tokens
  bool bad = false;
  for (int b = lo; b < hi; ++b) {
    const int raw_cached = p.cached_lens[b], raw_len = p.seq_lens[b];
    const int cached = max(0, min(raw_cached, most)), len = max(0, min(raw_len, most));
    bad |= cached != raw_cached || len != raw_len;
    s_seq[b] = make_int4(sum[0], sum[1], cached, len);
    sum[0] += max(len - cached, 0);
    sum[1] += max(blocks(len) - blocks(cached), 0);
    sum[2] += len;
  }
  int before[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    int incl = sum[k];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += v;
    }
    if (lane == 31) s_warp[k][warp] = incl;
    before[k] = incl - sum[k];
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kMapsThreads / 32; ++w)
#pragma unroll
    for (int k = 0; k < 3; ++k)
      if (w < warp) before[k] += s_warp[k][w];
  const bool first_block = blockIdx.x == 0;
  int keys = before[2];
  for (int b = lo; b < hi; ++b) {
    int4 x = s_seq[b];
    x.x += before[0];
    x.y += before[1];
    s_seq[b] = x;
    if (first_block) {
      p.cu_q[b] = min(x.x, p.rows);
      p.cu_k[b] = keys;
    }
    keys += x.w;
  }
  if (hi == p.batch && lo < hi) {  // one thread: the last run's
    const int total = before[0] + sum[0], taken = before[1] + sum[1];
    s_seq[p.batch] = make_int4(total, taken, 0, 0);
    if (first_block) {
      p.cu_q[p.batch] = min(total, p.rows);
      p.cu_k[p.batch] = keys;
      *p.taken = taken;
      if (total > p.rows) atomicOr(p.status, NVLLM_STATUS_BAD_SLOT);
    }
  }
  if (first_block && bad) atomicOr(p.status, NVLLM_STATUS_BAD_BLOCK);
  __syncthreads();

  auto fresh = [&](int k) { return k < p.n_free ? p.free_blocks[k] : -1; };
  const unsigned step = gridDim.x * kMapsThreads, start = blockIdx.x * kMapsThreads + tid;
  for (unsigned i = start; i < static_cast<unsigned>(p.batch) * p.width; i += step) {  // below 2^23
    const int b = i / p.width, col = i - b * p.width;
    const int4 x = s_seq[b];
    const int held = blocks(x.z);
    if (col >= held) p.block_tables[b * p.bt_stride + col] = col < blocks(x.w) ? fresh(x.y + col - held) : -1;
  }
  const int total = s_seq[p.batch].x;
  for (unsigned t = start; t < static_cast<unsigned>(p.rows); t += step) {
    int slot = -1;
    int64_t position = 0;
    if (static_cast<int>(t) < total) {
      int b = 0, end = p.batch;  // the last sequence that starts at t or before, so one that has a token here
      while (end - b > 1) {
        const int mid = (b + end) >> 1;
        if (s_seq[mid].x <= static_cast<int>(t)) b = mid;
        else end = mid;
      }
      const int4 x = s_seq[b];
      const int pos = x.z + static_cast<int>(t) - x.x, col = pos / kBlockSize, held = blocks(x.z);
      const int blk = col < held ? p.block_tables[b * p.bt_stride + col] : fresh(x.y + col - held);
      if (blk >= 0 && blk <= 0x7fffffff / kBlockSize - 1) slot = blk * kBlockSize + pos % kBlockSize;
      position = pos;
    }
    p.slots[t] = slot;
    p.positions[t] = position;
  }
}

}  // namespace nvllm

extern "C" int nvllm_step_maps(const int32_t* seq_lens, const int32_t* cached_lens, int32_t batch, int32_t* block_tables,
                               int64_t bt_row_stride, int32_t max_blocks, const int32_t* free_blocks, int32_t num_free,
                               int32_t* cu_seqlens_q, int32_t* cu_seqlens_k, int32_t* slot_mapping, int64_t* positions,
                               int64_t num_rows, int32_t* blocks_taken, void* stream) {
  using namespace nvllm;
  if (batch <= 0 || batch > kMapsMaxBatch)
    return fail(NVLLM_E_GEOMETRY, "step_maps: batch=%d outside 1 to %d", batch, kMapsMaxBatch);
  if (max_blocks <= 0 || bt_row_stride < max_blocks || num_free < 0)
    return fail(NVLLM_E_GEOMETRY, "step_maps: max_blocks=%d must be positive and within the row stride, num_free=%d not negative",
                max_blocks, num_free);
  if (static_cast<int64_t>(batch) * max_blocks * kBlockSize > 0x7fffffffLL || num_rows < 0 || num_rows > 0x7fffffffLL)
    return fail(NVLLM_E_GEOMETRY, "step_maps: batch=%d x max_blocks=%d tokens or num_rows=%lld do not fit 32 bits", batch, max_blocks,
                (long long)num_rows);
  if (!seq_lens || !cached_lens || !block_tables || !cu_seqlens_q || !cu_seqlens_k || !blocks_taken ||
      (num_free > 0 && !free_blocks) || (num_rows > 0 && (!slot_mapping || !positions)))
    return fail(NVLLM_E_NULL, "step_maps: NULL pointer argument");
  StepMapsParams p;
  p.status = status_word();
  if (!p.status) return fail(NVLLM_E_NO_DEVICE, "step_maps: no CUDA device is usable");
  p.seq_lens = seq_lens;
  p.cached_lens = cached_lens;
  p.batch = batch;
  p.block_tables = block_tables;
  p.bt_stride = bt_row_stride;
  p.width = max_blocks;
  p.free_blocks = free_blocks;
  p.n_free = num_free;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.slots = slot_mapping;
  p.positions = positions;
  p.rows = static_cast<int>(num_rows);
  p.taken = blocks_taken;
  const size_t smem = (static_cast<size_t>(batch) + 1) * sizeof(int4);
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {  // whatever this batch needs: the kernel's own arrays come on top of it
    const cudaError_t e = cudaFuncSetAttribute(step_maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kMapsMaxBatch + 1) * sizeof(int4));
    if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "step_maps: cannot reserve shared memory: %s", cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  // an entry and a row to a thread, as long as there are SMs: every block makes the sums itself
  const int64_t items = num_rows > static_cast<int64_t>(batch) * max_blocks ? num_rows : static_cast<int64_t>(batch) * max_blocks;
  const int64_t grid = std::min<int64_t>((items + kMapsThreads - 1) / kMapsThreads, 2ll * num_sms());
  return launch_kernel("step_maps", step_maps_kernel, dim3(static_cast<unsigned>(std::max<int64_t>(grid, 1))), dim3(kMapsThreads), smem,
                       static_cast<cudaStream_t>(stream), p);
}
