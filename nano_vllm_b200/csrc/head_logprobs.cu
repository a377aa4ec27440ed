// Log probabilities of given tokens and entropy from hidden states: the LM head's product whose epilogue is the softmax.
//
// logits = hidden [N, H] weight [V, H]^T are never written: a tile of 128 rows x up to 256 columns is accumulated in tensor
// memory by tcgen05 and reduced there to three numbers for each row (maximum, sum of exponentials, their sum times the
// logits: the statistics of token_logprobs), which a second launch joins over the vocabulary's tiles.
//
// Sums over H stay fp32, in a tensor core that cuts its running sum towards zero at every step of 16 products.  That is a systematic
// loss: at H = 4096 logits come out 3.2e-6 too small, log probabilities 2e-6 off.  Two things are done about it.  A product is cut
// after kChunk elements and the parts are added in registers.  And the logits' scale makes good what a step loses on average
// (kStepLoss, half a last place of a sum that is still on its way, measured at 64 to 5120 elements, products of either sign and of
// one): at H = 1024 logits are 1.0e-6 off on average without, 5e-8 with it, log probabilities 4.6e-7 and 1.9e-7, the entropy 8.4e-7
// and 1.2e-7 (relative, 512 rows of 151936); at 4096 4.6e-7 and 1.7e-7, 9.1e-7 and 1.5e-7; fp32 sums without a tensor core are 1.9e-7
// off at 1024.  Sums that lose nothing, such as those of one product, come out too large by what is made good: 9.5e-7 of a difference
// of logits at the most.  Parts of 512 elements would halve the loss too, at 1.28 times the time for 4096 x 1024 x 151936.
//
// What bounds it.  Many rows: the tensor cores, and then the power cap (4096 x 1024 x 151936 803 us, 1590 TFLOP/s, 908 in a long chain;
// 1000 x 4096 830-870; blocks of 128 rows by themselves, which feed the tensor cores twice the bytes, 1306 and 1248).  H below some
// 900: the reduction of a tile (4096 x 512 490 us of 393; tiles shared out evenly to the warps the same; 16 warps instead of 8 made
// 77 x 896 47.6 instead of 45.9).  Up to 128 rows: the weights' stream (one row of 1024 53.5 us, 5.8 TB/s; of 4096 197.6, 6.3), with as
// many stages as fit on their way (four: 54.8 and 200.8).
#include <algorithm>
#include <atomic>

#include "logprobs.cuh"
#include "prefill_tc.cuh"

namespace nvllm {
namespace hlp {
using namespace sm100;

// Two blocks of a cluster work as a pair on 256 rows (PAIR): each has half of the rows and half of the columns' weights in its
// shared memory, the first one's thread multiplies both with tcgen05 of two blocks, and each reduces its own rows.
constexpr int BM = 128, BN = 256, BK = 64;
constexpr int kChunk = 1024;
constexpr double kStepLoss = 1.5e-8;
// A stage holds what is loaded of a tile's rows and its columns for 64 elements of k.  The product reads 128 rows all the same:
// behind the loaded ones whatever follows, which ends in accumulator rows that nobody reads (the last stage's lie in the slack).
constexpr int CTRL_BYTES = 1024, RING_BYTES = 192 * 1024, SLACK_BYTES = BM * BK * 2;
constexpr int SMEM = CTRL_BYTES + RING_BYTES + SLACK_BYTES + 1024;  // + alignment
constexpr int TMEM_COLS = 512;  // two accumulators
constexpr int MAX_NST = 16;
enum Bar { FULL0 = 0, EMPTY0 = MAX_NST, ACC_FULL0 = 2 * MAX_NST, ACC_FREE0 = 2 * MAX_NST + 2, DRAIN = 2 * MAX_NST + 4, NUM_BARS };

template <bool PAIR, bool LONG>
struct Cfg {
  static constexpr int WARPS = 8, COLS = BN / (WARPS / 4);  // of the epilogue; columns of a thread
  static constexpr int THREADS = (WARPS + 4) * 32;          // registers come by fours of warps
  // registers at launch and as the groups share them: the parts of long sums are added in those of the epilogue
  static constexpr int REGS = 168, REGS_EPILOGUE = 216, REGS_OTHER = 72;
  static_assert(!LONG || WARPS * REGS_EPILOGUE + 4 * REGS_OTHER <= (WARPS + 4) * REGS, "no more than the block has");
};

#ifdef __CUDACC__
// The same place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// A tile load of one block of a pair whose bytes are counted by a barrier of either.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, uint32_t cluster_bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void umma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One arrival at the barrier of both blocks when the products issued so far are done.
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(static_cast<uint16_t>(3))
               : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void alloc_tmem(uint32_t dst) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(TMEM_COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, TMEM_COLS);
  }
}
template <bool PAIR>
__device__ __forceinline__ void dealloc_tmem(uint32_t addr) {
  if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(TMEM_COLS) : "memory");
  else tmem_dealloc(addr, TMEM_COLS);
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
#endif

struct Params {
  const int64_t* tokens;
  const float* temperatures;
  float scale;    // of the logits
  int rows, vocab;
  int bn;         // columns of a tile
  int mt, nt;     // tiles of rows and of columns
  int group, ng;  // column tiles that a unit of work has one after the other, and how many such groups
  int mb;         // row tiles whose units take turns
  int a_rows;     // rows of a tile that are loaded (of each block)
  int nst;        // stages
  int kb;         // blocks of 64 elements of a row
  int keep;       // a thread block has one row tile all along
  float4* partial;  // [slot][half][mt * 128]: maximum, sum, sum times logits
  float* given;     // [mt * 128]: logit of the row's token
  int* status;
};

struct Unit {
  int m, g;
};
__device__ __forceinline__ Unit unit_of(const Params& p, int i) {
  const int full = p.mb * p.ng, sb = i / full, r = i - sb * full, cnt = min(p.mb, p.mt - sb * p.mb);
  return {sb * p.mb + r % cnt, r / cnt};
}

template <bool PAIR, bool LONG>
__global__ void __launch_bounds__(Cfg<PAIR, LONG>::THREADS, 1)
    head_logprobs_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Params p) {
  using G = Cfg<PAIR, LONG>;
  constexpr int WARPS = G::WARPS, COLS = G::COLS, CTAS = PAIR ? 2 : 1;
  const int a_bytes = p.a_rows * BK * 2, stage_bytes = a_bytes + p.bn / CTAS * BK * 2, nst = p.nst;
  extern __shared__ unsigned char smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR ? blockIdx.x & 1 : 0;  // in the pair
  const int first_unit = blockIdx.x / CTAS, unit_step = gridDim.x / CTAS;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](int i) { return base + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + 512);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + 520);
  const uint32_t ring = base + CTRL_BYTES;
  if (tid == 0) {
    *abort_flag = 0;
    for (int i = 0; i < NUM_BARS; ++i) mbar_init(bar(i), i == ACC_FREE0 || i == ACC_FREE0 + 1 ? CTAS * WARPS : 1u);
    mbar_fence_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == WARPS + 1) alloc_tmem<PAIR>(smem_u32(tmem_slot));
  tc_fence_before();
  if constexpr (PAIR) cluster_sync();  // the other block's barriers are there
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  const int units = p.mt * p.ng, chunks = LONG ? (p.kb * BK + kChunk - 1) / kChunk : 1, per_chunk = LONG ? kChunk / BK : p.kb;

  if (warp >= WARPS) {
    if constexpr (LONG) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(G::REGS_OTHER));
    if (warp == WARPS) {
      // ------------------------------------------------------------------ TMA producer
      if (elect_one()) {
        const int b_rows = p.bn / CTAS;
        const uint32_t bytes = CTAS * stage_bytes;  // of both blocks: the first one's barriers count them
        int s = 0, use = 0;
        bool ok = true;
        for (int i = first_unit; i < units && ok; i += unit_step) {
          const Unit u = unit_of(p, i);
          for (int n = u.g * p.group; n < min((u.g + 1) * p.group, p.nt) && ok; ++n)
            for (int kb = 0; kb < p.kb; ++kb) {
              if (use > 0 && !(ok = wait_or_abort(bar(EMPTY0 + s), (use - 1) & 1, abort_flag))) break;
              const uint32_t dst = ring + s * stage_bytes;
              if (rank == 0) mbar_expect_tx(bar(FULL0 + s), bytes);
              if constexpr (PAIR) {
                const uint32_t full = map_to(bar(FULL0 + s), 0);
                tma_load_pair(dst, &map_a, full, kb * BK, 0, (u.m * 2 + rank) * BM);
                tma_load_pair(dst + a_bytes, &map_b, full, kb * BK, 0, n * p.bn + rank * b_rows);
              } else {
                tma_load_3d(dst, &map_a, bar(FULL0 + s), kb * BK, 0, u.m * BM);
                tma_load_3d(dst + a_bytes, &map_b, bar(FULL0 + s), kb * BK, 0, n * p.bn);
              }
              if (++s == nst) {
                s = 0;
                ++use;
              }
            }
        }
        // Neither a copy nor an arrival is in flight when the block (the pair) ends: the last products that read a stage arrive at both
        // blocks' barriers; where a wait ran out, the first block's barriers tell of the copies of both.
        auto uses = [&](int k) { return k < s ? use + 1 : use; };
        for (int k = 0; k < nst && ok; ++k)
          if (uses(k) > 0) ok = wait_or_abort(bar(EMPTY0 + k), (uses(k) - 1) & 1, abort_flag);
        if (!ok && rank == 0)
          for (int k = 0; k < nst; ++k)
            if (uses(k) > 0) (void)mbar_wait(bar(FULL0 + k), (uses(k) - 1) & 1);
      }
    } else if (warp == WARPS + 1 && rank == 0) {
      // ------------------------------------------------------------------ MMA issuer
      if (elect_one()) {
        const uint32_t idesc = umma_idesc(BM * CTAS, p.bn, 0, 0);
        const uint64_t desc0 = umma_desc(ring, 16, 1024);
        auto commit = [&](int i) {
          if constexpr (PAIR) commit_pair(bar(i));
          else umma_commit(bar(i));
        };
        int s = 0, use = 0, it = 0;
        bool ok = true;
        for (int i = first_unit; i < units && ok; i += unit_step) {
          const Unit u = unit_of(p, i);
          for (int n = u.g * p.group; n < min((u.g + 1) * p.group, p.nt) && ok; ++n)
            for (int c = 0; c < chunks && ok; ++c, ++it) {
              const int b = it & 1;
              if (it >= 2 && !(ok = wait_or_abort(bar(ACC_FREE0 + b), ((it >> 1) - 1) & 1, abort_flag))) break;
              tc_fence_after();
              const int first = c * per_chunk, last = min(first + per_chunk, p.kb);
              for (int kb = first; kb < last; ++kb) {
                if (!(ok = wait_or_abort(bar(FULL0 + s), use & 1, abort_flag))) break;
                tc_fence_after();
                const uint64_t da = desc0 + static_cast<uint64_t>((s * stage_bytes) >> 4), db = da + (a_bytes >> 4);
#pragma unroll
                for (int ks = 0; ks < BK / 16; ++ks) {
                  if constexpr (PAIR) umma_pair(tmem + b * BN, da + 2 * ks, db + 2 * ks, idesc, kb > first || ks > 0);
                  else umma_ss(tmem + b * BN, da + 2 * ks, db + 2 * ks, idesc, kb > first || ks > 0);
                }
                commit(EMPTY0 + s);
                if (++s == nst) {
                  s = 0;
                  ++use;
                }
              }
              if (ok) commit(ACC_FULL0 + b);
            }
        }
        if (!ok) {  // nothing may still be running on tensor memory when it is freed
          commit(DRAIN);
          (void)mbar_wait(bar(DRAIN), 0);
        }
      }
    }
  } else {
    if constexpr (LONG) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(G::REGS_EPILOGUE));
    // ------------------------------------------------------------------ epilogue: a row and COLS of the columns to a thread
    const int part = warp >> 2, r = rank * BM + (warp & 3) * 32 + lane;
    const uint32_t at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + part * COLS;
    const int64_t rows_padded = static_cast<int64_t>(p.mt) * BM * CTAS;
    LpSums sum{-FLT_MAX, 0.f, 0.f};
    int it = 0, slot = 0;
    int64_t row = -1;
    float c = 0.f;
    int64_t token = -1;
    bool ok = true, live = true;  // live: of the warp's rows there is one
    auto flush = [&]() { p.partial[(static_cast<int64_t>(slot) * (WARPS / 4) + part) * rows_padded + row] = make_float4(sum.m, sum.s, sum.t, 0.f); };
    auto free_acc = [&](int b) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (rank == 0) mbar_arrive(bar(ACC_FREE0 + b));
        else arrive_at(map_to(bar(ACC_FREE0 + b), 0));
      }
    };
    constexpr int W = LONG ? 16 : 32;  // columns at a time
    auto add = [&](float (&v)[W], int col, int n) {  // from column col of the vocabulary, of which the first n count
      if (n < W) {
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (k >= n) v[k] = -INFINITY;
      }
      float most = v[0];
#pragma unroll
      for (int k = 1; k < W - 1; k += 2) most = fmax3(most, v[k], v[k + 1]);
      most = fmaxf(most, v[W - 1]);
      sum.rescale(fmaxf(most, sum.m), c);
      const uint64_t minus_m = pack2(-sum.m, -sum.m), c2 = pack2(c, c);
      uint64_t s2 = 0, t2 = 0;
#pragma unroll
      for (int k = 0; k < W; k += 2) {
        float a, b, ya, yb;
        unpack2(add2(pack2(v[k], v[k + 1]), minus_m), ya, yb);
        const uint64_t y2 = pack2(max_nan(ya, -3e38f), max_nan(yb, -3e38f));
        unpack2(mul2(y2, c2), a, b);
        const uint64_t w2 = pack2(fast_exp2(a), fast_exp2(b));
        s2 = add2(s2, w2);
        t2 = fma2(w2, y2, t2);
      }
      float a, b;
      unpack2(s2, a, b);
      sum.s += a + b;
      unpack2(t2, a, b);
      sum.t += a + b;
      const int64_t d = token - col;
      if (d >= 0 && d < W && d < n) {
        float x = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k)
          if (k == d) x = v[k];
        p.given[row] = x;
      }
    };
    for (int i = first_unit; i < units && ok; i += unit_step) {
      const Unit u = unit_of(p, i);
      if (row < 0 || !p.keep) {
        slot = u.g;
        sum = {-FLT_MAX, 0.f, 0.f};
        row = static_cast<int64_t>(u.m) * (BM * CTAS) + r;
        live = row - lane < p.rows;
        token = row < p.rows ? p.tokens[row] : -1;
        if (token >= p.vocab) token = -1;
        c = (row < p.rows ? lp_inverse(p.temperatures, row) : 1.f) * p.scale * 1.4426950408889634f;
      }
      for (int n = u.g * p.group; n < min((u.g + 1) * p.group, p.nt) && ok; ++n) {
        const int first = n * p.bn + part * COLS, end = min(p.vocab, (n + 1) * p.bn) - first;  // columns of this thread
        if constexpr (!LONG) {
          const int b = it & 1;
          if (!(ok = wait_or_abort(bar(ACC_FULL0 + b), (it >> 1) & 1, abort_flag))) break;
          ++it;
          __syncwarp();
          tc_fence_after();
#pragma unroll 1
          for (int j = 0; j < end && j < COLS && live; j += 32) {
            uint32_t v[32];
            tmem_ld32(at + b * BN + j, v);
            tmem_wait_ld();
            float x[32];
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = __uint_as_float(v[k]);
            add(x, first + j, end - j);
          }
          free_acc(b);
        } else {
          float acc[COLS];
          for (int ch = 0; ch < chunks; ++ch, ++it) {
            const int b = it & 1;
            if (!(ok = wait_or_abort(bar(ACC_FULL0 + b), (it >> 1) & 1, abort_flag))) break;
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < COLS; j += W) {
              uint32_t v[W];
              tmem_ld16(at + b * BN + j, v);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < W; ++k) acc[j + k] = ch == 0 ? __uint_as_float(v[k]) : acc[j + k] + __uint_as_float(v[k]);
            }
            free_acc(b);
          }
          if (!ok) break;
#pragma unroll
          for (int j = 0; j < COLS; j += W) {
            if (j < end && live) {
              float x[W];
#pragma unroll
              for (int k = 0; k < W; ++k) x[k] = acc[j + k];
              add(x, first + j, end - j);
            }
          }
        }
      }
      if (!p.keep) flush();
    }
    if (p.keep && row >= 0) flush();
  }

  __syncwarp();
  pdl_trigger();
  tc_fence_before();
  if constexpr (PAIR) cluster_sync();  // neither block's memory is in use any more
  else __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(p.status, NVLLM_STATUS_TIMEOUT);
  if (warp == WARPS + 1) {
    tc_fence_after();
    dealloc_tmem<PAIR>(tmem);
  }
}

// Joins the partial statistics of `slots` slots for every row: a block has `wide` rows and deals a row's slots out to 256 / wide
// threads (one row to a block where there are few: 37 trips to memory one after the other in each of eight threads a row cost 6 us).
struct JoinParams {
  const float4* partial;
  const float* given;
  const int64_t* tokens;
  const float* temperatures;
  float scale;
  int rows, vocab, slots, wide;  // slots: halves counted
  int64_t rows_padded;
  float *logprobs, *entropy;
  int* status;
};
constexpr int kJoinThreads = 256;

__global__ void __launch_bounds__(kJoinThreads) join_kernel(const JoinParams p) {
  __shared__ float s_sums[3][kJoinThreads];
  const int tid = threadIdx.x, part = tid / p.wide, parts = kJoinThreads / p.wide;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * p.wide + tid % p.wide;
  const bool live = row < p.rows;
  const float inv_t = (live ? lp_inverse(p.temperatures, row) : 1.f) * p.scale, c = inv_t * 1.4426950408889634f;
  const int64_t token = live ? p.tokens[row] : -1;
  pdl_prologue();
  LpSums sum{-FLT_MAX, 0.f, 0.f};
  float given = 0.f;
  if (live) {
    if (part == 0 && token >= 0 && token < p.vocab) given = p.given[row];
    constexpr int U = 8;
    for (int k = part; k < p.slots; k += U * parts) {
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u * parts < p.slots) v[u] = p.partial[static_cast<int64_t>(k + u * parts) * p.rows_padded + row];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (k + u * parts < p.slots) sum.join(v[u].x, v[u].y, v[u].z, c);
    }
  }
  for (int n = parts / 2; n > 0; n /= 2) {
    s_sums[0][tid] = sum.m;
    s_sums[1][tid] = sum.s;
    s_sums[2][tid] = sum.t;
    __syncthreads();
    if (part < n) {
      const int o = tid + n * p.wide;
      sum.join(s_sums[0][o], s_sums[1][o], s_sums[2][o], c);
    }
    __syncthreads();
  }
  if (part == 0 && live) sum.results(row, token, given, inv_t, sum.log_z(), p.vocab, p.logprobs, p.entropy, p.status);
}

// How a problem is laid out over the multiprocessors.
struct Plan {
  int pair, bn, mt, nt, group, ng, mb, kb, keep, grid, slots, a_rows, nst;
  int64_t rows_padded, bytes;
};
static Plan plan_of(int rows, int hidden, int vocab, int sms) {
  Plan pl;
  pl.pair = rows > BM;
  const int bm = pl.pair ? 2 * BM : BM, workers = std::max(1, pl.pair ? sms / 2 : sms);
  pl.kb = (hidden + BK - 1) / BK;
  pl.mt = (rows + bm - 1) / bm;
  pl.a_rows = pl.pair ? BM : std::min(BM, (rows + 7) / 8 * 8);
  // The widest tile that leaves the worker with most tiles as few columns as any, in steps that tcgen05 of one block and of two take.
  // A pair's are not below 192 columns, where a tile's operands take longer to come than their product: 4096 x 1024 x 151936 in tiles of 128
  // columns 1138 us, 160 984, 192 908, 224 925, 256 931 (calls one after the other, at the power cap).  Up to 128 rows the weights are most of
  // what is loaded: 77 x 896 in tiles of 128 columns 50.2 us, 176 49.6, 208 49.2, 256 53.8.
  int64_t least = 0;
  pl.bn = BN;
  for (int bn = BN; bn >= (pl.pair ? 192 : 128); bn -= pl.pair ? 32 : 16) {
    const int64_t tiles = static_cast<int64_t>(pl.mt) * ((vocab + bn - 1) / bn), cost = (tiles + workers - 1) / workers * bn;
    if (bn == BN || cost < least) least = cost, pl.bn = bn;
  }
  pl.nt = (vocab + pl.bn - 1) / pl.bn;
  pl.nst = std::min(MAX_NST, RING_BYTES / ((pl.a_rows + pl.bn / (pl.pair ? 2 : 1)) * BK * 2));
  pl.keep = pl.mt <= workers && workers % pl.mt == 0;
  pl.group = 1;
  while (!pl.keep && pl.group < 16 && static_cast<int64_t>(pl.mt) * ((pl.nt + 2 * pl.group - 1) / (2 * pl.group)) >= 48ll * workers) pl.group *= 2;
  // no more than 64 MB of partial statistics, as long as there is a longer group
  while (!pl.keep && pl.group < pl.nt && 2ll * ((pl.nt + pl.group - 1) / pl.group) * pl.mt * bm * 16 > (64 << 20)) pl.group *= 2;
  pl.ng = (pl.nt + pl.group - 1) / pl.group;
  pl.mb = pl.keep ? pl.mt : static_cast<int>(std::min<int64_t>(pl.mt, std::max<int64_t>(1, std::min<int64_t>(16, (32ll << 20) / (bm * 2ll * hidden)))));
  pl.grid = static_cast<int>(std::min<int64_t>(workers, static_cast<int64_t>(pl.mt) * pl.ng)) * (pl.pair ? 2 : 1);
  const int parts = hidden > kChunk ? Cfg<false, true>::WARPS / 4 : Cfg<false, false>::WARPS / 4;
  pl.slots = parts * (pl.keep ? std::min(workers / pl.mt, pl.ng) : pl.ng);
  pl.rows_padded = static_cast<int64_t>(pl.mt) * bm;
  pl.bytes = pl.slots * pl.rows_padded * 16 + pl.rows_padded * 4;
  return pl;
}

// What makes good the mean loss of sums over `hidden` elements: of every part its own steps', the first of which has nothing to lose.
// (All as if they were full ones: logits of 1472 elements 1.4e-7 too large on average.)
static float scale_of(int64_t hidden) {
  double lost = 0;
  for (int64_t at = 0; at < hidden; at += kChunk) {
    const int64_t n = std::min<int64_t>(kChunk, hidden - at);
    lost += static_cast<double>(n) * static_cast<double>((n + 15) / 16 - 1);
  }
  return static_cast<float>(1 + kStepLoss * lost / static_cast<double>(hidden));
}

static int check(int64_t rows, int64_t hidden, int64_t vocab) {
  if (rows < 0 || rows > (1 << 24) || vocab <= 0 || vocab > (1 << 21) || hidden <= 0 || hidden > 65536 || hidden % 8)
    return fail(NVLLM_E_GEOMETRY, "head_logprobs: rows=%lld hidden=%lld (a multiple of 8) vocab=%lld not supported", (long long)rows, (long long)hidden,
                (long long)vocab);
  return NVLLM_OK;
}

}  // namespace hlp
}  // namespace nvllm

extern "C" int64_t nvllm_head_logprobs_workspace_bytes(int64_t rows, int64_t hidden, int64_t vocab) {
  using namespace nvllm;
  if (const int e = hlp::check(rows, hidden, vocab)) return e;
  if (rows == 0) return 0;
  const int sms = num_sms();
  return hlp::plan_of(static_cast<int>(rows), static_cast<int>(hidden), static_cast<int>(vocab), sms > 0 ? sms : 148).bytes;
}

extern "C" int nvllm_head_logprobs(const void* hidden_states, int64_t hidden_row_stride, const void* weight, int64_t weight_row_stride,
                                   const int64_t* tokens, const float* temperatures, int64_t rows, int64_t hidden, int64_t vocab,
                                   float* logprobs, float* entropy, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace nvllm;
  if (const int e = hlp::check(rows, hidden, vocab)) return e;
  if (rows == 0) return NVLLM_OK;
  if (!hidden_states || !weight || !tokens || !logprobs || !entropy) return fail(NVLLM_E_NULL, "head_logprobs: NULL pointer argument");
  if (hidden_row_stride < hidden || weight_row_stride < hidden) return fail(NVLLM_E_GEOMETRY, "head_logprobs: a row stride is smaller than a row");
  auto off = [](const void* q, size_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
  if (!aligned16(hidden_states) || !aligned16(weight) || hidden_row_stride % 8 || weight_row_stride % 8 || off(tokens, 8) || off(temperatures, 4) ||
      off(logprobs, 4) || off(entropy, 4))
    return fail(NVLLM_E_ALIGN, "head_logprobs: rows must be 16-byte aligned, the other pointers aligned to their elements");
  const int sms = num_sms();
  int* status = status_word();
  if (!status || sms <= 0) return fail(NVLLM_E_NO_DEVICE, "head_logprobs: no CUDA device is usable");
  const hlp::Plan pl = hlp::plan_of(static_cast<int>(rows), static_cast<int>(hidden), static_cast<int>(vocab), sms);
  if (!workspace || workspace_bytes < pl.bytes)
    return fail(NVLLM_E_WORKSPACE, "head_logprobs: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)pl.bytes);
  if (!aligned16(workspace)) return fail(NVLLM_E_ALIGN, "head_logprobs: the workspace must be 16-byte aligned");
  CUtensorMap a, b;
  if (!sm100::make_tmap_3d(&a, hidden_states, hidden, 1, rows, hidden_row_stride, hidden_row_stride, pl.a_rows)) return NVLLM_E_CUDA;
  if (!sm100::make_tmap_3d(&b, weight, hidden, 1, vocab, weight_row_stride, weight_row_stride, pl.pair ? pl.bn / 2 : pl.bn)) return NVLLM_E_CUDA;
  const bool is_long = hidden > hlp::kChunk;
  using Kernel = decltype(&hlp::head_logprobs_kernel<false, false>);
  static const Kernel kernels[2][2] = {{hlp::head_logprobs_kernel<false, false>, hlp::head_logprobs_kernel<false, true>},
                                       {hlp::head_logprobs_kernel<true, false>, hlp::head_logprobs_kernel<true, true>}};
  // All forms are made ready by the first call on a device, so that later ones can be captured whatever their sizes.
  static std::atomic<bool> ready[64];
  static std::atomic<int> registers[2][2];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !ready[dev]) {
    for (int k = 0; k < 4; ++k) {
      cudaError_t e = cudaFuncSetAttribute(kernels[k / 2][k % 2], cudaFuncAttributeMaxDynamicSharedMemorySize, hlp::SMEM);
      if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "head_logprobs: cannot reserve shared memory: %s", cudaGetErrorString(e));
      cudaFuncAttributes attr;
      if ((e = cudaFuncGetAttributes(&attr, kernels[k / 2][k % 2])) != cudaSuccess)
        return fail(NVLLM_E_CUDA, "head_logprobs: %s", cudaGetErrorString(e));
      registers[k / 2][k % 2] = attr.numRegs;
    }
    if (dev >= 0 && dev < 64) ready[dev] = true;
  }
  // a block with fewer registers than its groups share would wait for them without end
  if (is_long && registers[pl.pair][is_long] < hlp::Cfg<false, true>::REGS)
    return fail(NVLLM_E_CUDA, "head_logprobs: compiled to %d registers, %d needed", registers[pl.pair][is_long].load(), hlp::Cfg<false, true>::REGS);
  hlp::Params p{};
  p.tokens = tokens;
  p.temperatures = temperatures;
  p.scale = hlp::scale_of(hidden);
  p.rows = static_cast<int>(rows);
  p.vocab = static_cast<int>(vocab);
  p.bn = pl.bn;
  p.mt = pl.mt;
  p.nt = pl.nt;
  p.group = pl.group;
  p.ng = pl.ng;
  p.mb = pl.mb;
  p.a_rows = pl.a_rows;
  p.nst = pl.nst;
  p.kb = pl.kb;
  p.keep = pl.keep;
  p.partial = static_cast<float4*>(workspace);
  p.given = reinterpret_cast<float*>(p.partial + pl.slots * pl.rows_padded);
  p.status = status;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.grid);
  cfg.blockDim = dim3(is_long ? hlp::Cfg<false, true>::THREADS : hlp::Cfg<false, false>::THREADS);
  cfg.dynamicSmemBytes = hlp::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pl.pair ? 2 : 1;
  const cudaError_t launched = cudaLaunchKernelEx(&cfg, kernels[pl.pair][is_long], a, b, p);
  count_launch();
  if (launched != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(NVLLM_E_CUDA, "head_logprobs launch: %s", cudaGetErrorString(launched));
  }
  int wide = 1;
  while (wide < 32 && rows > 4ll * sms * wide) wide *= 2;
  const hlp::JoinParams j{p.partial, p.given, tokens, temperatures, p.scale, p.rows, p.vocab, pl.slots, wide, pl.rows_padded, logprobs, entropy, status};
  return launch_kernel("head_logprobs", hlp::join_kernel, dim3(static_cast<unsigned>((rows + wide - 1) / wide)), dim3(hlp::kJoinThreads), 0, st, j);
}
