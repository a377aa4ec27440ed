// Paged GQA decode attention over the 8-bit cache (fp8.cuh), one query token per sequence, for sm_100a.
//
//   out[b,h] = sum_t softmax_t(scale q[b,h] . K[t,h/G]) V[t,h/G],  K, V = code * scale of the token's group and head
//
// The step variant also does what store_kvcache_fp8 does for the one new token of every sequence.
//
// Bound by the cached bytes, half of a bf16 cache's: 128 sequences of 1024-8192 tokens (32 / 8 heads of 128) 185 us, 6.4 TB/s
// (bf16: 363), 180 with nothing computed; launch after launch, with the power cap on the clocks, 204.  The launch is cut as the bf16 decode's is (decode_paged.cu): all sequences' work units
// in one list, an equal stretch of it to each of two resident blocks per SM, partial results of sequences that a cut
// divides merged by the last block to arrive.  What differs is what a tile costs:
//   * A warp of its own loads: table entries, tiles by TMA (a box for every warp's tile that holds a token), scales.  When the
//     four others did that themselves, with cp.async, they spent half of their instructions on it; a barrier of the block
//     for every unit instead was slower (128 sequences 199 -> 214 us, loading warp 184; 60 of 100-1024 21.5, 23.3, 18.3,
//     all before merges of few parts had code of their own).
//   * K codes go from shared memory to registers 16 bytes a lane and become f16 pairs there (cvt, exact, two cycles).  The four
//     codes of a word are columns k = 2 tig .. and k = 2 tig + 8 .. of one m16n8k16 product: the order of the summed index
//     is free, the query's columns follow it.
//   * V codes go through ldmatrix.trans as pairs of neighbouring columns: a register then holds two columns of two tokens,
//     one byte permutation away from (token, token) pairs of either column, rows gid and gid + 8 of V^T.
//   * q is f16 too, scaled by a power of two to 2^14 <= max |q| < 2^15, so that it keeps all its bits down to 2^-29 of the
//     largest.  The group's K scale multiplies the fp32 scores.  P, times 2^12 and the group's V scale over the warp's running
//     unit, is rounded to f16: the sums O are held in that unit, which follows the scales (see `unit`).  2^12 takes P to
//     f16's upper end: weights down to 2^-24 of the largest keep all its bits, and what those below lose is 2^-35 of the largest
//     each, in all 2^-18 of it over 131072 keys.  (Without it the keys that shared a warp with a first key 18 nats above them, 32768
//     to a sequence, were lost: the result came out at 86 % of its value.)
//   * 16 tokens share a scale, so a group lies in one warp's tile: the step variant's warp that streams the new token has
//     its whole group at hand, codes the row, codes the rows before it anew where the scale grows, and writes them back.
//
// Small batches are bound by trips one after the other: lengths and split (0.7 us), table entry, tiles, the products of a tile
// (0.7), flush (0.6), arrival (0.8), merge (of two to four parts 1.5 us by short code of its own, by that for any number 3).  The
// first three run ahead of the wait for the previous kernel and are verified behind it (a sequence of 317 tokens 7.1 -> 6.7 us
// in a chain, 60 of 100-1024 23.1 -> 22.4, two of 100000 (head_dim 64) 20 -> 18.6; with all that came later 5.5, 17.6 and 18.2).
#include "fp8.cuh"
#include "sm100.cuh"

namespace nvllm {

// Workspace: as nvllm_decode_paged's.  [arrival counters][partials O][partials (max, sum)]
constexpr int kFp8CounterSlots = 16384;
constexpr int64_t kFp8CounterBytes = static_cast<int64_t>(kFp8CounterSlots) * 4;
constexpr int kFp8MaxCtas = 1024;

struct DecodeFp8Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  unsigned char* k_cache;  // written by the step variant, as the scales are
  unsigned char* v_cache;
  float* k_scale;
  float* v_scale;
  const int32_t* ctx_lens;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  __nv_bfloat16* out;
  int64_t out_stride;
  int batch, hq, hkv, g;
  float scale_log2e;
  int64_t num_blocks;
  const __nv_bfloat16* k_new;  // step variant
  int64_t k_new_stride;
  const __nv_bfloat16* v_new;
  int64_t v_new_stride;
  const int32_t* slot_mapping;
  int n_ranges;
  unsigned int* counters;  // [batch * hkv], zero between launches
  float* ws_o;             // [n_ranges + batch][hq][D]
  float* ws_ml;            // [n_ranges + batch][hq][2] = (running max in log2 units, sum)
  int* status;
};

template <int D_, int TT_, int NST_, int NW_, int BLOCKS_>
struct DecodeFp8Cfg {
  static constexpr int D = D_, TT = TT_, NST = NST_, NW = NW_, BLOCKS = BLOCKS_;  // blocks to an SM
  static constexpr int UNIT = NW * TT;  // tokens of a work unit
  static constexpr int MT = TT / 16;    // groups of a warp's tile
  static constexpr int CPR = D / 16;    // 16-byte pieces of a row
  static constexpr int TILE_BYTES = TT * D;       // a warp's part of a unit
  static constexpr int UNIT_BYTES = UNIT * D;
  static constexpr int STAGE_BYTES = 2 * UNIT_BYTES;
  static constexpr int RING_BYTES = NST * STAGE_BYTES;
  static constexpr int UNIT_GROUPS = UNIT / kScaleGroup;
  static constexpr int SCALE_BYTES = 2 * UNIT_GROUPS * 4;  // of a stage: K's, V's
  static constexpr int OFF_SCALES = RING_BYTES;
  static constexpr int OFF_MERGE = OFF_SCALES + NST * SCALE_BYTES;
  static constexpr int OROW = D + 4;    // floats of a head's row: sums, maximum, sum; heads written together lie in different banks
  static constexpr int OFF_CTRL = OFF_MERGE + NW * 8 * OROW * 4;  // barriers, then a few words
  static constexpr int SMEM = OFF_CTRL + 2 * NST * 8 + (NST + NW + 3 + 2) * 4;
  static constexpr int NTHREADS = (NW + 1) * 32;  // and a warp that loads
  static constexpr int KS = D / 16;  // products of a group's scores, and of its share of O
  static_assert(TT % kScaleGroup == 0 && kBlockSize % UNIT == 0 && (MT & (MT - 1)) == 0 && MT <= 4, "whole groups, units within a block");
  static_assert(TILE_BYTES % 1024 == 0 && OFF_MERGE % 16 == 0, "a warp's tile starts where the swizzle does");
  static_assert(BLOCKS * (SMEM + 1024) <= 228 * 1024, "as many blocks to an SM");
};

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ld_shared_f32(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_f32(uint32_t a, float v) { asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(a), "f"(v) : "memory"); }
// Where TMA's swizzle puts piece c of row r of a tile (128-byte rows; or 64-byte ones, two to a line).
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int r, int c) {
  return r * D + ((c ^ (D == 128 ? r & 7 : r >> 1 & 3)) << 4);
}
// The token of row i < 8 of a matrix operand.  Neighbouring rows of K are read together, a half of 64 bytes each: at D = 128
// tokens four apart lie in different banks.  The order is free as long as V's is the same.
template <int D>
__device__ __forceinline__ int token_of_row(int i) {
  return D == 128 ? (i >> 1) | (i & 1) << 2 : i;
}

struct Fp8Cursor {  // the sequence a block is working in: index, global index of its first unit, units, length
  int b, first, units, ctx;
  int slot;  // step variant: of the new token, -1: nothing is stored
};
struct Fp8Cut {  // a sequence whose units lie in several ranges: n of them, from r_first on
  int b, r_first, n;
};

// Cost of a streamed unit over the cost of a merged partial (decode_paged.cu: the same trade).  With 4, 8, 16, 32: one sequence of
// 8192 tokens (32 / 8 heads of 128) 9.9, 9.6, 8.8, 9.4 us, two of 2000 (16 / 8) 7.4, 7.5, 6.6, 6.6, two of 110000 (14 / 2 of 64) 20, 16.6,
// 16.1, 16.1.
constexpr float kFp8SplitBalance = 16.f;
// What goes on P, and how far V's scales may go from the unit of O: their product stays in f16, which ends at 2^16.
constexpr float kFp8Weight = 0x1p12f, kFp8UnitUp = 8.f, kFp8UnitDown = 4.f;

template <class C, bool STEP>
__global__ void __launch_bounds__(C::NTHREADS, C::BLOCKS)
decode_fp8_kernel(const DecodeFp8Params p, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v) {
  constexpr int D = C::D, TT = C::TT, NST = C::NST, NW = C::NW, UNIT = C::UNIT, MT = C::MT, NT = NW * 32;
  constexpr int QUADS = D / 4, GROUPS = NT / QUADS;  // lanes that hold a head four columns each; such groups in a block
  constexpr int PIECES = D / 8;                      // lanes that hold a bf16 row, eight values each
  constexpr unsigned ALL = 0xffffffffu;
  extern __shared__ __align__(1024) unsigned char smem[];
  // in the dynamic part, which would start 1024 bytes later behind any other: two blocks to an SM need all but 900 bytes
  uint64_t* s_full = reinterpret_cast<uint64_t*>(smem + C::OFF_CTRL);
  uint64_t* s_free = s_full + NST;
  int *s_row = reinterpret_cast<int*>(s_free + NST), *s_scan = s_row + NST;
  int *s_start = s_scan + NW, *s_last_arrival = s_start + 3;

  pdl_trigger();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < NST; ++i) {
      sm100::mbar_init(smem_u32(s_full + i), 2);  // the tiles; the scales
      sm100::mbar_init(smem_u32(s_free + i), NW);
    }
    sm100::mbar_fence_init();
    sm100::prefetch_tmap(&tmap_k);
    sm100::prefetch_tmap(&tmap_v);
  }
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int kvh = blockIdx.x % p.hkv;
  const int range = blockIdx.x / p.hkv;
  const int ctx_cap = p.max_blocks * kBlockSize;
  auto length_of = [&](int b) { return max(0, min(p.ctx_lens[b], ctx_cap)); };
  auto units_of = [](int ctx) { return (ctx + UNIT - 1) / UNIT; };
  auto write_zeros = [&](int b) {  // empty context: defined output, no cache access
    if (b % p.n_ranges != range) return;
    uint4* dst = reinterpret_cast<uint4*>(p.out + b * p.out_stride + static_cast<int64_t>(kvh * p.g) * D);
    for (int i = 0; i < p.g * D / 8; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
  };

  // ---- 1. units per sequence, block-wide scan, this block's range of the unit list ------
  const bool loader = warp == NW;
  const int per_thread = loader ? 0 : (p.batch + NT - 1) / NT;
  const int b_lo = min(tid * per_thread, p.batch), b_hi = min(b_lo + per_thread, p.batch);
  int total, n_ranges, per_range, longer, u0, u1, len_lo;
  int2* seqs = reinterpret_cast<int2*>(smem + C::OFF_MERGE);  // ahead: first unit and length of every sequence
  static_assert(NT * 8 <= C::OFF_CTRL - C::OFF_MERGE, "room for them until the first merge");
  auto split = [&](bool ahead) {  // whether this block has a range
    int local = 0;
    len_lo = 0;
    for (int b = b_lo; b < b_hi; ++b) {
      const int c = ahead ? max(0, min(__ldcg(p.ctx_lens + b), ctx_cap)) : length_of(b);
      if (b == b_lo) len_lo = c;
      local += units_of(c);
    }
    int incl = local;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(ALL, incl, d);
      if (lane >= d) incl += v;
    }
    if (lane == 31 && !loader) s_scan[warp] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    const int excl = before + incl - local;
    if (ahead && !loader) seqs[tid] = make_int2(excl, len_lo);
    // No more ranges than units, and where sequences are few no more than balance the two costs of a cut: a range streams
    // total / n units and a sequence's merge reads n / batch partials.
    n_ranges = max(1, min(min(p.n_ranges, total), static_cast<int>(sqrtf(kFp8SplitBalance * total * p.batch))));
    // Two units one after the other take less than a merge, three and four do not: one sequence of 200 tokens (16 / 8 heads of 128) 4.35 us,
    // cut 5.3; 317 5.3, 5.35; 512 6.5, 5.35; its step 5.0, 5.6; 6.0, 5.6; 7.15, 5.75.  Of 512, 600, 900 (14 / 2 of 64) 4.1, 5.05; 5.0, 5.15; 5.95,
    // 5.2.
    if (p.batch == 1 && total <= 2) n_ranges = 1;
    if (range >= n_ranges || total == 0) return false;  // block-uniform
    per_range = total / n_ranges, longer = total - per_range * n_ranges;  // the first `longer` ranges hold one more
    u0 = range * per_range + min(range, longer), u1 = u0 + per_range + (range < longer ? 1 : 0);
    if (local > 0 && excl <= u0 && u0 < excl + local) {  // the one thread whose sequences hold unit u0
      int first = excl;
      for (int b = b_lo;; ++b) {
        const int len = b == b_lo ? len_lo : length_of(b), n = units_of(len);
        if (u0 < first + n) {
          s_start[0] = b;
          s_start[1] = first;
          s_start[2] = len;
          break;
        }
        first += n;
      }
    }
    __syncthreads();
    return true;
  };
  // Batches of a sequence to a thread at most: the split is made, and the first units' table entries are read and their tiles
  // brought to L2, while the previous kernel still runs.  It may change lengths and tables: when it is done they are read
  // again, in one trip, and if one has changed the split is made anew.  What is read before the wait goes round L1, is held
  // to the bounds of the table and the cache, and serves the guess alone.
  int n_listed = 0, listed_blk = -1;  // the loading warp: units whose entries are known, one to a lane
  bool mine;
#pragma unroll 1
  for (bool ahead = p.batch <= NT;; ahead = false) {
    if (!ahead) pdl_wait();
    mine = split(ahead);
    if (!ahead) break;
    const int32_t* at = nullptr;
    if (mine && loader) {
      n_listed = min(u1 - u0, NST);
      int row = -1;
      if (lane < n_listed) {
        const int u = u0 + lane;
        int b = s_start[0];
        while (b + 1 < p.batch && u >= seqs[b].x + units_of(seqs[b].y)) ++b;
        const int unit0 = (u - seqs[b].x) * UNIT;
        at = p.block_tables + b * p.bt_stride + unit0 / kBlockSize;
        listed_blk = __ldcg(at);
        if (listed_blk >= 0 && listed_blk < p.num_blocks) row = listed_blk * kBlockSize + unit0 % kBlockSize;
      }
#pragma unroll 1
      for (int k0 = 0; k0 < n_listed * 2 * NW; k0 += 32) {
        const int k = k0 + lane, from = __shfl_sync(ALL, row, min(k / (2 * NW), 31));
        if (k < n_listed * 2 * NW && from >= 0) sm100::tma_prefetch_3d(k & 1 ? &tmap_v : &tmap_k, 0, kvh, from + k % (2 * NW) / 2 * TT);
      }
    }
    pdl_wait();
    const bool changed = (!loader && tid < p.batch && length_of(tid) != len_lo) || (at && *at != listed_blk);
    if (!__syncthreads_or(changed)) break;
    n_listed = 0;
  }
  for (int b = b_lo; b < b_hi; ++b)
    if (length_of(b) == 0) write_zeros(b);
  if (!mine) return;

  auto range_of = [&](int u) {  // the range that holds global unit u
    const int split = longer * (per_range + 1);
    return u < split ? u / (per_range + 1) : longer + (u - split) / per_range;
  };

  auto slot_of = [&](int b) { return STEP ? p.slot_mapping[b] : -1; };
  auto seek = [&](Fp8Cursor& c, int u) {  // u < total, so c.b stays inside the batch
    if (u < c.first + c.units) return;
    do {
      c.first += c.units;
      ++c.b;
      c.ctx = length_of(c.b);
      c.units = units_of(c.ctx);
    } while (u >= c.first + c.units);
    c.slot = slot_of(c.b);
  };

  const int n_units = u1 - u0;
  const uint32_t ring = smem_u32(smem), scale_ring = ring + C::OFF_SCALES;
  auto full = [&](int i) { return smem_u32(s_full + i % NST); };
  auto free = [&](int i) { return smem_u32(s_free + i % NST); };
  auto sync_warps = [&]() { asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory"); };  // of those that compute
  Fp8Cursor cc;
  cc.b = s_start[0];
  cc.first = s_start[1];
  cc.ctx = s_start[2];
  cc.units = units_of(cc.ctx);
  cc.slot = slot_of(cc.b);
  int bad = 0;

  // ---- 2. the loading warp: units by TMA (a box to a warp's tile that holds a token), their scales a group to a lane ----
  if (loader) {
    const bool of_v = lane >= C::UNIT_GROUPS;
    const float* scales = of_v ? p.v_scale : p.k_scale;
    auto block_at = [&](int j) -> int64_t {  // of the range's j-th unit; the cursor goes along
      seek(cc, u0 + j);
      const int64_t blk = j < n_listed ? __shfl_sync(ALL, listed_blk, j)
                                       : p.block_tables[cc.b * p.bt_stride + (u0 + j - cc.first) * UNIT / kBlockSize];
      if (blk >= 0 && blk < p.num_blocks) return blk;
      bad |= NVLLM_STATUS_BAD_BLOCK;
      return p.num_blocks;  // rows behind the cache: zeros
    };
    auto scale_of = [&](int64_t blk, int unit0) {
      if (blk >= p.num_blocks || lane >= 2 * C::UNIT_GROUPS) return 0.f;
      return scales[(blk * p.hkv + kvh) * kGroups + unit0 % kBlockSize / kScaleGroup + lane % C::UNIT_GROUPS];
    };
    int64_t blk = block_at(0);
    float scale = scale_of(blk, (u0 - cc.first) * UNIT);
    int j = 0;
#pragma unroll 1
    for (; j < n_units; ++j) {
      const int unit0 = (u0 + j - cc.first) * UNIT;
      if (j >= NST && !__all_sync(ALL, sm100::mbar_wait(free(j), (j / NST - 1) & 1))) {
        bad |= NVLLM_STATUS_TIMEOUT;
        break;
      }
      const int row = static_cast<int>(blk * kBlockSize + unit0 % kBlockSize);
      if (lane == 0) {
        const uint32_t dst = ring + j % NST * C::STAGE_BYTES;
        const int tiles = min((cc.ctx - unit0 + TT - 1) / TT, NW);
        sm100::mbar_expect_tx(full(j), tiles * 2 * C::TILE_BYTES);
#pragma unroll 1
        for (int w = 0; w < tiles; ++w) {
          sm100::tma_load_3d(dst + w * C::TILE_BYTES, &tmap_k, full(j), 0, kvh, row + w * TT);
          sm100::tma_load_3d(dst + C::UNIT_BYTES + w * C::TILE_BYTES, &tmap_v, full(j), 0, kvh, row + w * TT);
        }
        s_row[j % NST] = row;
      }
      // the next unit's entry and scales, on their way while this one's tiles are
      const float scale_now = scale;
      if (j + 1 < n_units) {
        blk = block_at(j + 1);
        scale = scale_of(blk, (u0 + j + 1 - cc.first) * UNIT);
      }
      if (lane < 2 * C::UNIT_GROUPS) st_shared_f32(scale_ring + j % NST * C::SCALE_BYTES + lane * 4, scale_now);
      __syncwarp();
      if (lane == 0) sm100::mbar_arrive(full(j));
    }
    // No copy is in flight when the block ends, whether or not the others have waited for it.
#pragma unroll 1
    for (int i = max(j - NST, 0); i < j; ++i)
      if (!sm100::mbar_wait(full(i), (i / NST) & 1)) bad |= NVLLM_STATUS_TIMEOUT;
    if (bad && lane == 0) atomicOr(p.status, bad);
    return;
  }

  // ---- the query: lane (gid, tig) holds columns 16 (tig + 4 j) .. + 15 of head gid ------------
  constexpr int QW = D / 8;  // words of them
  auto load_q = [&](uint32_t (&dst)[QW], int b) {
    const uint4* row = reinterpret_cast<const uint4*>(p.q + b * p.q_stride + static_cast<int64_t>(kvh * p.g + gid) * D);
#pragma unroll
    for (int j = 0; j < D / 64; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = gid < p.g ? row[2 * (tig + 4 * j) + i] : make_uint4(0, 0, 0, 0);
        uint32_t* to = dst + 8 * j + 4 * i;
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
      }
  };
  uint32_t qb[QW];        // f16 pairs: word 2 ks + e is the B operand of product ks
  float qk0 = 0.f, qk1 = 0.f;  // what takes the products of heads 2 tig and 2 tig + 1 to log2 units, K's scale apart
  auto take_q = [&](const uint32_t (&raw)[QW]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < QW; ++i) m = max_finite2(m, raw[i]);
    m = max(m & 0xffffu, m >> 16);
    m = max(m, __shfl_xor_sync(ALL, m, 1));
    m = max(m, __shfl_xor_sync(ALL, m, 2));
    const int e = max(static_cast<int>(m >> 7), 20) - 127;  // 2^e <= max |q| < 2^(e + 1)
    const float f = power_of_two(14 - e);
#pragma unroll
    for (int i = 0; i < QW; ++i) qb[i] = pack_f16x2(__uint_as_float(raw[i] << 16) * f, __uint_as_float(raw[i] & 0xffff0000u) * f);
    const float back = p.scale_log2e * power_of_two(e - 14);
    qk0 = __shfl_sync(ALL, back, 8 * tig);
    qk1 = __shfl_sync(ALL, back, 8 * tig + 4);
  };

  // ---- 3. the other warps: a tile of every unit -------------------------------------------------
  const uint32_t warp_tile = ring + warp * C::TILE_BYTES, warp_scales = scale_ring + warp * MT * 4;
  const int64_t row_bytes = static_cast<int64_t>(p.hkv) * D;
  const bool is_v = lane >= 16;
  const int sub = (lane & 15) / PIECES, piece = lane % PIECES;
  // Step variant: the new token's row of a sequence, K in the lower half of the warp, V in the upper, eight values a lane.
  auto load_new = [&](int b) {
    const __nv_bfloat16* src = (is_v ? p.v_new + b * p.v_new_stride : p.k_new + b * p.k_new_stride) + kvh * D + piece * 8;
    return sub == 0 ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
  };
  uint4 new_row = make_uint4(0, 0, 0, 0), next_row = new_row;
  uint32_t qn[QW];  // the next sequence's query, and its row, fetched early
  load_q(qn, cc.b);
  if (STEP) new_row = load_new(cc.b);
  take_q(qn);
  int qn_b = min(cc.b + 1, p.batch - 1);
  load_q(qn, qn_b);
  if (STEP) next_row = load_new(qn_b);

  float o[C::KS][4];     // columns 16 c + 2 gid (and + 1 in [2], [3]) of heads 2 tig ([0], [2]) and 2 tig + 1, in units of `unit`
  float m0, m1, l0, l1;  // heads 2 tig and 2 tig + 1
  // What O is held in (the same for all lanes of the warp): a group's P goes into its product times vscale / unit.  It is the
  // largest scale of the first tile, changed where a tile's largest is more than 8 times larger or 4 times smaller, so that P,
  // up to 2^12, stays below f16's end and loses two bits of its range at most; not below 2^-60 of what it has been, which keeps
  // O finite whatever the scales; and not below 2^-114, so that it is normal when the 2^12 is taken off: smaller scales,
  // subnormal ones too, leave P to f16's lower end.
  constexpr float least_unit = 0x1p-114f;
  float unit, most_unit;
  auto reset_state = [&]() {
#pragma unroll
    for (int c = 0; c < C::KS; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    m0 = m1 = -INFINITY;
    l0 = l1 = 0.f;
    unit = least_unit;
    most_unit = 0.f;
  };
  reset_state();

  constexpr int OROW = C::OROW;
  float* sm_o = reinterpret_cast<float*>(smem + C::OFF_MERGE);  // [NW][8][OROW]
  auto add_scaled = [](float4& acc, const float4& v, float f) {
    acc.x += v.x * f;
    acc.y += v.y * f;
    acc.z += v.z * f;
    acc.w += v.w * f;
  };
  auto write_quad = [&](int b, int h, int d4, const float4& acc, float L) {
    const float inv = L > 0.f ? 1.f / L : L;  // no key: zeros; a sum that is NaN stays one
    *reinterpret_cast<uint2*>(p.out + b * p.out_stride + static_cast<int64_t>(kvh * p.g + h) * D + d4 * 4) =
        make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  };

  Fp8Cut cut0{}, cut1{};  // this range's sequences that other ranges share
  int n_cut = 0;

  // Leaves sequence cc.b: merges the NW warps' states and writes the output row or a partial.
  auto flush = [&]() {
#pragma unroll
    for (int sh = 4; sh <= 16; sh <<= 1) {
      l0 += __shfl_xor_sync(ALL, l0, sh);
      l1 += __shfl_xor_sync(ALL, l1, sh);
    }
    const float by = unit * (1.f / kFp8Weight);
    sync_warps();  // the previous merge has been read by everyone
#pragma unroll
    for (int c = 0; c < C::KS; ++c) {
      float* dst = sm_o + (warp * 8 + 2 * tig) * OROW + c * 16 + 2 * gid;
      *reinterpret_cast<float2*>(dst) = make_float2(o[c][0] * by, o[c][2] * by);
      *reinterpret_cast<float2*>(dst + OROW) = make_float2(o[c][1] * by, o[c][3] * by);
    }
    if (gid == 0) {
      float* dst = sm_o + (warp * 8 + 2 * tig) * OROW + D;
      *reinterpret_cast<float2*>(dst) = make_float2(m0, l0);
      *reinterpret_cast<float2*>(dst + OROW) = make_float2(m1, l1);
    }
    int r_first = range, n_parts = 1;  // ranges that hold a piece of this sequence
    if (cc.first < u0 || cc.first + cc.units > u1) {
      r_first = range_of(cc.first);
      n_parts = range_of(cc.first + cc.units - 1) - r_first + 1;
    }
    sync_warps();
    for (int quad = tid; quad < p.g * QUADS; quad += NT) {  // four columns of a head per thread
      const int h = quad / QUADS, d4 = quad % QUADS;
      float m[NW], mm = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        m[w] = sm_o[(w * 8 + h) * OROW + D];
        mm = fmaxf(mm, m[w]);
      }
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = m[w] == -INFINITY ? 0.f : fast_exp2(m[w] - mm);
        const float4 v = *reinterpret_cast<const float4*>(sm_o + (w * 8 + h) * OROW + d4 * 4);
        L += sm_o[(w * 8 + h) * OROW + D + 1] * f;
        add_scaled(acc, v, f);
      }
      if (n_parts == 1) {
        write_quad(cc.b, h, d4, acc, L);
      } else {
        // partial slot range + b: strictly increasing along the (range, sequence) pieces of the list
        const int64_t row = static_cast<int64_t>(range + cc.b) * p.hq + kvh * p.g + h;
        *reinterpret_cast<float4*>(p.ws_o + row * D + d4 * 4) = acc;
        if (d4 == 0) *reinterpret_cast<float2*>(p.ws_ml + row * 2) = make_float2(mm, L);
      }
    }
    if (n_parts > 1) {  // block-uniform
      if (n_cut == 0) cut0 = {cc.b, r_first, n_parts};
      else cut1 = {cc.b, r_first, n_parts};
      ++n_cut;
    }
  };

  // Merges the partials of a cut sequence, all of which are in the workspace, and writes its rows: QUADS lanes take a head,
  // four columns each, and the statistics of a part each; sixteen parts to a trip; lane groups left over split the parts.
  auto merge_cut = [&](const Fp8Cut& c) {
    constexpr int AHEAD = 16;
    static_assert(AHEAD <= QUADS, "a lane for each part's statistics");
    const int group = tid / QUADS, gl = tid % QUADS;
    const int n_split = max(1, GROUPS / p.g);
    for (int h0 = 0; h0 < p.g; h0 += GROUPS) {
      const bool narrow = p.g < GROUPS;
      const int split = narrow ? group / p.g : 0, head = narrow ? group % p.g : min(h0 + group, p.g - 1);
      const bool active = narrow ? split < n_split : h0 + group < p.g;
      const int64_t row0 = static_cast<int64_t>(c.r_first + c.b) * p.hq + kvh * p.g + head;
      auto row_of = [&](int j) { return __ldcg(reinterpret_cast<const float4*>(p.ws_o + (row0 + static_cast<int64_t>(j) * p.hq) * D) + gl); };
      float mm = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      auto rebase = [&](float m_new) {
        const float keep = mm == -INFINITY ? 0.f : fast_exp2(mm - m_new);
        L *= keep;
        acc.x *= keep;
        acc.y *= keep;
        acc.z *= keep;
        acc.w *= keep;
        mm = m_new;
      };
#pragma unroll 1
      for (int j0 = 0; j0 < c.n; j0 += AHEAD * n_split) {  // block-uniform; a group's parts are split + n_split * k
        float4 rows[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int j = j0 + k * n_split + split;
          if (active && j < c.n) rows[k] = row_of(j);
        }
        const int mine = j0 + gl * n_split + split;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (active && gl < AHEAD && mine < c.n)
          ml = __ldcg(reinterpret_cast<const float2*>(p.ws_ml + (row0 + static_cast<int64_t>(mine) * p.hq) * 2));
        float m_new = fmaxf(mm, ml.x);
#pragma unroll
        for (int sh = QUADS / 2; sh > 0; sh >>= 1) m_new = fmaxf(m_new, __shfl_xor_sync(ALL, m_new, sh));
        rebase(m_new);
        const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m_new);
        float sum = ml.y * f;
#pragma unroll
        for (int sh = QUADS / 2; sh > 0; sh >>= 1) sum += __shfl_xor_sync(ALL, sum, sh);
        L += sum;
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const float fk = __shfl_sync(ALL, f, k, QUADS);
          if (active && j0 + k * n_split + split < c.n) add_scaled(acc, rows[k], fk);
        }
      }
      if (n_split > 1) {  // block-uniform
        float* patch = sm_o + group * (D + 4);
        if (active && split > 0) {
          *reinterpret_cast<float4*>(patch + gl * 4) = acc;
          if (gl == 0) *reinterpret_cast<float2*>(patch + D) = make_float2(mm, L);
        }
        sync_warps();
        if (active && split == 0)
          for (int k = 1; k < n_split; ++k) {
            const float* other = sm_o + (group + k * p.g) * (D + 4);
            const float2 ml = *reinterpret_cast<const float2*>(other + D);
            rebase(fmaxf(mm, ml.x));
            const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mm);
            L += ml.y * f;
            add_scaled(acc, *reinterpret_cast<const float4*>(other + gl * 4), f);
          }
        sync_warps();
      }
      if (active && split == 0) write_quad(c.b, head, gl, acc, L);
    }
    if (tid == 0) p.counters[c.b * p.hkv + kvh] = 0u;  // ready for the next launch
  };

  // The same of a few parts, which is what a batch's sequences are cut into as a rule: a thread its columns of all of them.  A merge
  // is the last thing that a block does and runs once, so its instructions come from L2, at 25 cycles each: short code it is.
  constexpr int FEW = 4;
  auto merge_few = [&](const Fp8Cut& c) {
    const int64_t row0 = static_cast<int64_t>(c.r_first + c.b) * p.hq + kvh * p.g;
#pragma unroll 1
    for (int x = tid; x < p.g * QUADS; x += NT) {
      const int64_t row = row0 + x / QUADS;
      float2 ml[FEW];
      float4 v[FEW], acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float top = -INFINITY, L = 0.f;
#pragma unroll
      for (int j = 0; j < FEW; ++j) {
        const int64_t at = row + static_cast<int64_t>(min(j, c.n - 1)) * p.hq;
        ml[j] = __ldcg(reinterpret_cast<const float2*>(p.ws_ml + at * 2));
        v[j] = __ldcg(reinterpret_cast<const float4*>(p.ws_o + at * D) + x % QUADS);
      }
#pragma unroll
      for (int j = 0; j < FEW; ++j) {
        if (j >= c.n) ml[j] = make_float2(-INFINITY, 0.f);
        top = fmaxf(top, ml[j].x);
      }
#pragma unroll
      for (int j = 0; j < FEW; ++j) {
        if (j >= c.n) continue;
        const float f = ml[j].x == -INFINITY ? 0.f : fast_exp2(ml[j].x - top);  // no maximum but a sum: NaN, which zero times it stays
        L += ml[j].y * f;
        add_scaled(acc, v[j], f);
      }
      write_quad(c.b, x / QUADS, x % QUADS, acc, L);
    }
    if (tid == 0) p.counters[c.b * p.hkv + kvh] = 0u;  // ready for the next launch
  };

  for (int i = 0;; ++i) {
    const int u = u0 + i;
    if (i == n_units || u >= cc.first + cc.units) {  // block-uniform: the range leaves sequence cc.b
      flush();
      if (i == n_units) break;
      seek(cc, u);
      reset_state();
      if (qn_b != cc.b) {  // empty sequences in between
        load_q(qn, cc.b);
        if (STEP) next_row = load_new(cc.b);
      }
      take_q(qn);
      new_row = next_row;
      qn_b = min(cc.b + 1, p.batch - 1);
      load_q(qn, qn_b);
      if (STEP) next_row = load_new(qn_b);
    }
    // A wait that ran out: nothing more is waited for or stored, and no stage is given back, so that the loading warp stops too; but all
    // barriers that the other warps count on are met.  (A vote here, to skip the tiles too, costs 3 % of the launch.)
    if (!(bad & NVLLM_STATUS_TIMEOUT) && !sm100::mbar_wait(full(i), (i / NST) & 1)) bad |= NVLLM_STATUS_TIMEOUT;
    const int t0 = (u - cc.first) * UNIT + warp * TT;
    if (t0 >= cc.ctx) {
      if (lane == 0 && !(bad & NVLLM_STATUS_TIMEOUT)) sm100::mbar_arrive(free(i));
      continue;
    }
    const uint32_t kbase = warp_tile + (i % NST) * C::STAGE_BYTES, vbase = kbase + C::UNIT_BYTES;
    const uint32_t scales = warp_scales + (i % NST) * C::SCALE_BYTES;

    const int r = cc.ctx - 1 - t0, r0 = r & ~(kScaleGroup - 1);  // the newest token's row of the tile, the first one of its group
    bool fresh = STEP && r < TT && cc.slot >= 0;
    if (fresh) {  // its place by the table, too
      fresh = cc.slot == s_row[i % NST] + warp * TT + r && cc.slot < p.num_blocks * kBlockSize;
      if (!fresh) bad |= NVLLM_STATUS_BAD_SLOT;
      fresh = !__any_sync(ALL, !fresh || (bad & NVLLM_STATUS_TIMEOUT));
    }
    if (fresh) {  // the new token's row: to the tile and to the cache, its group with it
      const uint4 x = new_row;
      uint32_t most = max_finite2(max_finite2(max_finite2(max_finite2(0, x.x), x.y), x.z), x.w);
      most = max(most & 0xffffu, most >> 16);
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(ALL, most, d));
      const uint32_t scale_smem = scales + (is_v ? C::UNIT_GROUPS * 4 : 0) + (r0 / kScaleGroup) * 4;
      const float old = ld_shared_f32(scale_smem);
      const int e = r > r0 ? max(exponent_for(most), exponent_of(old)) : exponent_for(most);
      const float now = power_of_two(e), inv = power_of_two(-e);
      const uint32_t tile = is_v ? vbase : kbase;
      unsigned char* to = (is_v ? p.v_cache : p.k_cache) + (static_cast<int64_t>(cc.slot) - r) * row_bytes + kvh * D + piece * 8;
      auto in_tile = [&](int row) { return tile + tile_offset<D>(row, piece >> 1) + (piece & 1) * 8; };
      if (r > r0 && now != old) {
        const float ratio = old * inv;
#pragma unroll 1
        for (int row = r0 + sub; row < r; row += 16 / PIECES) {
          uint2 c = ld_shared8(in_tile(row));
          c = make_uint2(recode4(c.x, ratio), recode4(c.y, ratio));
          st_shared8(in_tile(row), c);
          *reinterpret_cast<uint2*>(to + row * row_bytes) = c;
        }
      }
      if (sub == 0) {
        const uint2 c = make_uint2(encode4(make_uint2(x.x, x.y), inv), encode4(make_uint2(x.z, x.w), inv));
        st_shared8(in_tile(r), c);
        *reinterpret_cast<uint2*>(to + r * row_bytes) = c;
      }
      sm100::fence_proxy_async();  // TMA writes here again
      __syncwarp();
      if ((lane & 15) == 0) {
        st_shared_f32(scale_smem, now);
        const int64_t slot = cc.slot;
        (is_v ? p.v_scale : p.k_scale)[(slot / kBlockSize * p.hkv + kvh) * kGroups + slot % kBlockSize / kScaleGroup] = now;
      }
      __syncwarp();
    }

    const bool tail = t0 + TT > cc.ctx;
    if (tail) {  // V rows behind the end hold anything: zeros, which their weights leave what they are
      for (int x = (cc.ctx - t0) * C::CPR + lane; x < TT * C::CPR; x += 32)
        st_shared16(vbase + tile_offset<D>(x / C::CPR, x % C::CPR), make_uint4(0, 0, 0, 0));
      sm100::fence_proxy_async();
      __syncwarp();
    }

    // S^T = K Q^T, in log2 units
    float s[MT][4], vs[MT], most_vs = 0.f;
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      s[mt][0] = s[mt][1] = s[mt][2] = s[mt][3] = 0.f;
      float odd[4] = {0.f, 0.f, 0.f, 0.f};  // every other product: two chains instead of one
#pragma unroll
      for (int j = 0; j < D / 64; ++j) {
        const int ra = mt * 16 + token_of_row<D>(gid);
        const uint4 a = ld_shared16(kbase + tile_offset<D>(ra, tig + 4 * j)), b = ld_shared16(kbase + tile_offset<D>(ra + 8, tig + 4 * j));
        const uint32_t wa[4] = {a.x, a.y, a.z, a.w}, wb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int w = 0; w < 4; ++w)
          mma_f16_16816(w & 1 ? odd : s[mt], f16x2_of_low(wa[w]), f16x2_of_low(wb[w]), f16x2_of_high(wa[w]),
                        f16x2_of_high(wb[w]), qb[8 * j + 2 * w], qb[8 * j + 2 * w + 1]);
      }
      s[mt][0] += odd[0], s[mt][1] += odd[1], s[mt][2] += odd[2], s[mt][3] += odd[3];
      const float ks = ld_shared_f32(scales + mt * 4);
      vs[mt] = t0 + mt * 16 < cc.ctx ? ld_shared_f32(scales + (C::UNIT_GROUPS + mt) * 4) : 0.f;  // a group past the end: whatever is there
      most_vs = fmaxf(most_vs, vs[mt]);
      const float f0 = qk0 * ks, f1 = qk1 * ks;
      s[mt][0] = __fmul_rn(s[mt][0], f0);  // rounded here: the largest minus the maximum is zero, however large the scores are
      s[mt][1] = __fmul_rn(s[mt][1], f1);
      s[mt][2] = __fmul_rn(s[mt][2], f0);
      s[mt][3] = __fmul_rn(s[mt][3], f1);
      if (tail) {
        const int tr = t0 + mt * 16 + token_of_row<D>(gid);
        if (tr >= cc.ctx) s[mt][0] = s[mt][1] = -INFINITY;
        if (tr + 8 >= cc.ctx) s[mt][2] = s[mt][3] = -INFINITY;
      }
      mx0 = fmaxf(mx0, fmaxf(s[mt][0], s[mt][2]));
      mx1 = fmaxf(mx1, fmaxf(s[mt][1], s[mt][3]));
    }
#pragma unroll
    for (int sh = 4; sh <= 16; sh <<= 1) {
      mx0 = fmaxf(mx0, __shfl_xor_sync(ALL, mx0, sh));
      mx1 = fmaxf(mx1, __shfl_xor_sync(ALL, mx1, sh));
    }
    const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
    float alpha0 = fast_exp2(m0 - mn0), alpha1 = fast_exp2(m1 - mn1);
    l0 *= alpha0;
    l1 *= alpha1;
    if (most_vs > unit * kFp8UnitUp || (most_vs * kFp8UnitDown < unit && unit > least_unit && most_vs > 0.f)) {
      const float next = fminf(fmaxf(fmaxf(most_vs, most_unit * 0x1p-60f), least_unit), kLargestUnit), change = next != unit ? unit / next : 1.f;
      alpha0 *= change;
      alpha1 *= change;
      unit = next;
      most_unit = fmaxf(most_unit, next);
    }
    const float per_unit = 1.f / unit;
    m0 = mn0;
    m1 = mn1;
    uint32_t pb[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      s[mt][0] = fast_exp2(s[mt][0] - mn0);
      s[mt][1] = fast_exp2(s[mt][1] - mn1);
      s[mt][2] = fast_exp2(s[mt][2] - mn0);
      s[mt][3] = fast_exp2(s[mt][3] - mn1);
      l0 += s[mt][0] + s[mt][2];  // per-lane partial sums; reduced over the token lanes at the flush
      l1 += s[mt][1] + s[mt][3];
      const float f = mul_subnormal(vs[mt], per_unit) * kFp8Weight;
      pb[mt][0] = movmatrix_trans(pack_f16x2(s[mt][0] * f, s[mt][1] * f));
      pb[mt][1] = movmatrix_trans(pack_f16x2(s[mt][2] * f, s[mt][3] * f));
    }
    if (__any_sync(ALL, alpha0 != 1.f || alpha1 != 1.f)) {
#pragma unroll
      for (int c = 0; c < C::KS; ++c) {
        o[c][0] *= alpha0;
        o[c][1] *= alpha1;
        o[c][2] *= alpha0;
        o[c][3] *= alpha1;
      }
    }

    // O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int c = 0; c < C::KS; c += 2) {
        const int r = mt * 16 + (lane & 8) + token_of_row<D>(lane & 7);
        uint32_t v[4];  // tokens 0-7 and 8-15 of columns 16 c .., then of 16 (c + 1) ..
        ldmatrix_x4_trans(v[0], v[1], v[2], v[3], vbase + tile_offset<D>(r, c + (lane >> 4)));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t lo = __byte_perm(v[2 * k], 0, 0x3120), hi = __byte_perm(v[2 * k + 1], 0, 0x3120);
          mma_f16_16816(o[c + k], f16x2_of_low(lo), f16x2_of_high(lo), f16x2_of_low(hi), f16x2_of_high(hi), pb[mt][0], pb[mt][1]);
        }
      }
    }
    __syncwarp();  // everything of the unit is in registers
    if (lane == 0 && !(bad & NVLLM_STATUS_TIMEOUT)) sm100::mbar_arrive(free(i));
  }
  bad = __reduce_or_sync(ALL, bad);
  if (bad && lane == 0) atomicOr(p.status, bad);
  if (n_cut == 0) return;  // block-uniform
  sync_warps();            // every thread's partials are written
  if (tid < n_cut) {
    const Fp8Cut& c = tid == 0 ? cut0 : cut1;
    unsigned int arrived;  // releases the block's partials (the barrier ordered them before), acquires the others'
    asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                 : "=r"(arrived) : "l"(p.counters + c.b * p.hkv + kvh) : "memory");
    s_last_arrival[tid] = arrived == static_cast<unsigned int>(c.n - 1);
  }
  sync_warps();
#pragma unroll 1
  for (int k = 0; k < n_cut; ++k) {
    if (!s_last_arrival[k]) continue;
    const Fp8Cut c = k == 0 ? cut0 : cut1;
    if (c.n <= FEW) merge_few(c);
    else merge_cut(c);
  }
}

// ---- host side -------------------------------------------------------------------------

template <class C>
static int launch_decode_fp8(const DecodeFp8Params& p, cudaStream_t stream) {
  CUtensorMap mk, mv;
  const uint64_t slots = static_cast<uint64_t>(p.num_blocks) * kBlockSize;
  if (!sm100::make_tmap_codes(&mk, p.k_cache, C::D, p.hkv, slots, C::TT) || !sm100::make_tmap_codes(&mv, p.v_cache, C::D, p.hkv, slots, C::TT))
    return NVLLM_E_CUDA;
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    for (auto kernel : {decode_fp8_kernel<C, false>, decode_fp8_kernel<C, true>}) {
      const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
      if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "decode_fp8: cannot reserve %d bytes of shared memory: %s", C::SMEM, cudaGetErrorString(e));
    }
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return launch_kernel("decode_fp8", p.k_new ? decode_fp8_kernel<C, true> : decode_fp8_kernel<C, false>,
                       dim3(static_cast<unsigned>(p.n_ranges * p.hkv)), dim3(C::NTHREADS), C::SMEM, stream, p, mk, mv);
}

struct Fp8Cache {
  void *k, *v;
  float *k_scale, *v_scale;
};

static int decode_fp8_common(const char* who, const void* q, int64_t q_row_stride, const void* k_new, int64_t k_new_row_stride,
                             const void* v_new, int64_t v_new_row_stride, const int32_t* slot_mapping, bool with_store,
                             const Fp8Cache& cache, const int32_t* context_lens, const int32_t* block_tables, int64_t bt_row_stride,
                             int32_t max_blocks, void* out, int64_t out_row_stride, int32_t batch, int32_t num_q_heads,
                             int32_t num_kv_heads, int32_t head_dim, float scale, int64_t num_blocks, void* workspace,
                             int64_t workspace_bytes, void* stream) {
  const int64_t need = nvllm_decode_workspace_bytes(batch, max_blocks, num_q_heads, num_kv_heads, head_dim);
  if (need < 0) return static_cast<int>(need);
  if (!(scale >= 0.f && scale < INFINITY)) return fail(NVLLM_E_GEOMETRY, "%s: scale must be finite and not negative", who);
  if (batch == 0) return NVLLM_OK;
  const int rc = check_fp8_planes(who, cache.k, cache.v, cache.k_scale, cache.v_scale, num_kv_heads, head_dim, num_blocks);
  if (rc) return rc;
  if (!q || !context_lens || !block_tables || !out) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", who);
  const int64_t qrow = static_cast<int64_t>(num_q_heads) * head_dim, kvrow = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (q_row_stride < qrow || out_row_stride < qrow || bt_row_stride < max_blocks)
    return fail(NVLLM_E_GEOMETRY, "%s: a row stride is smaller than its row", who);
  if (q_row_stride % 8 || out_row_stride % 8 || !aligned16(q) || !aligned16(out))
    return fail(NVLLM_E_ALIGN, "%s: q/out pointers and row strides must be 16-byte aligned", who);
  if (with_store) {
    if (!k_new || !v_new || !slot_mapping) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", who);
    if (k_new_row_stride < kvrow || v_new_row_stride < kvrow)
      return fail(NVLLM_E_GEOMETRY, "%s: key/value row stride smaller than Hkv*D", who);
    if (k_new_row_stride % 8 || v_new_row_stride % 8 || !aligned16(k_new) || !aligned16(v_new))
      return fail(NVLLM_E_ALIGN, "%s: key/value pointers and row strides must be 16-byte aligned", who);
  }
  if (!workspace || workspace_bytes < need)
    return fail(NVLLM_E_WORKSPACE, "%s: workspace of %lld bytes needed, %lld given", who, (long long)need,
                (long long)(workspace ? workspace_bytes : 0));
  if (!aligned16(workspace)) return fail(NVLLM_E_ALIGN, "%s: workspace must be 16-byte aligned", who);
  DecodeFp8Params p;
  p.status = status_word();
  if (!p.status) return fail(NVLLM_E_NO_DEVICE, "%s: no CUDA device is usable", who);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_row_stride;
  p.k_cache = static_cast<unsigned char*>(cache.k);
  p.v_cache = static_cast<unsigned char*>(cache.v);
  p.k_scale = cache.k_scale;
  p.v_scale = cache.v_scale;
  p.ctx_lens = context_lens;
  p.block_tables = block_tables;
  p.bt_stride = bt_row_stride;
  p.max_blocks = max_blocks;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_row_stride;
  p.batch = batch;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.g = num_q_heads / num_kv_heads;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.num_blocks = num_blocks;
  p.k_new = with_store ? static_cast<const __nv_bfloat16*>(k_new) : nullptr;
  p.k_new_stride = k_new_row_stride;
  p.v_new = with_store ? static_cast<const __nv_bfloat16*>(v_new) : nullptr;
  p.v_new_stride = v_new_row_stride;
  p.slot_mapping = slot_mapping;
  auto ranges_for = [&](int ctas) { return ctas / num_kv_heads > 1 ? ctas / num_kv_heads : 1; };
  auto ranges_of = [&](int blocks) {
    const int ctas = blocks * num_sms();
    return ranges_for(ctas > 0 && ctas <= kFp8MaxCtas ? ctas : kFp8MaxCtas);
  };
  const int64_t rows = (static_cast<int64_t>(ranges_for(kFp8MaxCtas)) + batch) * num_q_heads;
  p.counters = static_cast<unsigned int*>(workspace);
  p.ws_o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kFp8CounterBytes);
  p.ws_ml = p.ws_o + rows * head_dim;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  using Wide = DecodeFp8Cfg<128, 32, 3, 4, 2>;
  using Narrow = DecodeFp8Cfg<64, 64, 2, 4, 2>;
  p.n_ranges = ranges_of(head_dim == 128 ? Wide::BLOCKS : Narrow::BLOCKS);
  return head_dim == 128 ? launch_decode_fp8<Wide>(p, st) : launch_decode_fp8<Narrow>(p, st);
}

}  // namespace nvllm

extern "C" int nvllm_decode_paged_fp8(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                      const float* k_scale, const float* v_scale, const int32_t* context_lens,
                                      const int32_t* block_tables, int64_t bt_row_stride, int32_t max_blocks, void* out,
                                      int64_t out_row_stride, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                      int32_t head_dim, float scale, int64_t num_blocks, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const nvllm::Fp8Cache cache = {const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<float*>(k_scale),
                                 const_cast<float*>(v_scale)};
  return nvllm::decode_fp8_common("decode_paged_fp8", q, q_row_stride, nullptr, 0, nullptr, 0, nullptr, false, cache, context_lens,
                                  block_tables, bt_row_stride, max_blocks, out, out_row_stride, batch, num_q_heads, num_kv_heads,
                                  head_dim, scale, num_blocks, workspace, workspace_bytes, stream);
}

extern "C" int nvllm_decode_step_fp8(const void* q, int64_t q_row_stride, const void* key, int64_t key_row_stride,
                                     const void* value, int64_t value_row_stride, const int32_t* slot_mapping, void* k_cache,
                                     void* v_cache, float* k_scale, float* v_scale, const int32_t* context_lens,
                                     const int32_t* block_tables, int64_t bt_row_stride, int32_t max_blocks, void* out,
                                     int64_t out_row_stride, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                                     int32_t head_dim, float scale, int64_t num_blocks, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  return nvllm::decode_fp8_common("decode_step_fp8", q, q_row_stride, key, key_row_stride, value, value_row_stride, slot_mapping,
                                  true, {k_cache, v_cache, k_scale, v_scale}, context_lens, block_tables, bt_row_stride, max_blocks,
                                  out, out_row_stride, batch, num_q_heads, num_kv_heads, head_dim, scale, num_blocks, workspace,
                                  workspace_bytes, stream);
}
