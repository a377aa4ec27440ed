// Varlen causal GQA prefill over the 8-bit cache (fp8.cuh) on the 5th-generation tensor cores, head_dim 64 or 128.
//
//   query i of a sequence with Lq new tokens of Lk sees keys j <= i + Lk - Lq;  K, V = code * scale of the token's group
//
// Tiles of 128 query rows (128 / n tokens x n heads that share a KV head) and 64 keys, four groups of scales:
//   * S = Q K^T with the codes as they come by TMA (kind::f8f6f4).  A row of Q, scaled by a power of two to 128 <= max < 256, is
//     the sum of two e4m3 numbers: the nearest, and what is left of bf16's eight bits, which has four at most.  Exact down to
//     2^-10 of the row's largest value, below that within 2^-17 of it.  Two products at twice the rate of a 16-bit one: the
//     same time, and no key has to be converted.
//   * The K scale of a group and the row's power of two enter the multiply-add in front of the exponential, four factors a tile.
//   * O += P V in f16 (kind::f16): P from TMEM, 2^8 to 2^15 at a row's largest score, rounded to f16: weights down to 2^-22 of the
//     largest keep all its bits, those below lose 2^-33 of it each.  V's codes become f16 once a tile, by the warps that also
//     write results, times the group's scale over the unit that O is held in: the largest scale of an item's first tile,
//     changed (and O with it) where a tile's largest is more than 2^7 times larger or 2^14 times smaller, which keeps every
//     V / unit an f16 number; not below 2^-60 of what it has been, which keeps O finite whatever the scales.  Exact for scales
//     that are powers of two, two more roundings to f16 for others.
//   * Keys past the end: their scores are masked, their V rows converted to zeros whatever the codes are.
//
// Twelve warps, two blocks to an SM for the whole launch: 0-3 softmax (thread = query row), 4-7 query rows in, V conversion and
// results out, 8 = TMA of the query rows, K and the scales, 9 = MMA issuer, 10 = TMA of V.  The three warp groups trade registers at
// start-up; 11 works out the items, one ahead.  Items (query tile of a sequence, head group) are ordered by their key tiles,
// most first, over all sequences, and dealt out in turn, there and back again, so that all blocks have about the same to do; no
// counter in memory, so nothing is shared by launches.  Where there are two blocks or more to an item (few new tokens behind a
// long prefix) an item's keys go to several of them (SPLIT), and prefill_fp8_join sums the parts up from the workspace.
//
// 4 x 4096 tokens (16 heads over 8 of 128) at full clocks: 299 us, 920 TFLOP/s, where scores are nearly flat, 353 where they spread by
// 2.2 nats with long tails; 12 sequences of 100-2000 tokens behind 256-4096 (14 over 2 of 64) 217 us.  Bound by the chain scores -
// softmax - P - product of a block, of which two to an SM overlap: of the 353 and 217, leaving out V's conversion saves 40 and 20, rescaling
// O 27 and 15, the exponentials 18 and 14; the tensor cores are busy 41 % of the time.
#include <algorithm>

#include "fp8.cuh"
#include "prefill_tc.cuh"
#include "sm100.cuh"

namespace nvllm {
using namespace sm100;

namespace f8 {
constexpr int BM = 128, BN = 64, KST = 2;
constexpr int MAX_BATCH = 1024;  // sequences of a launch
constexpr int NTHREADS = 384;
constexpr int REGS_LAUNCH = 80, REGS_SOFTMAX = 136, REGS_ROWS = 64, REGS_OTHER = 40;
static_assert(128 * (REGS_SOFTMAX + REGS_ROWS + REGS_OTHER) <= NTHREADS * REGS_LAUNCH, "register pool of a block");
constexpr int TMEM_COLS = 256, TMEM_O = 128;  // S / P buffers [0,64) and [64,128), O [128,256)
// Log2 units: P is 2^8 where a score is the maximum in use, which is kept until one is 2^7.9 times larger; f16 goes to 2^16.  (P from 1
// on, and 2^14, lost all that 131072 keys 18 nats below a first one have.)  Where a row outgrows its maximum, its warp's other rows go
// to theirs too.  4 x 4096 tokens (16 heads over 8 of 128, scores of 2.2 nats), one call after the other: 366 us; rows each for itself
// 380; 2^7 370, 2^5 371, 2^14 355.  (2^14 for an item's first 512 keys alone is 361, and loses 2^-26 of the largest on each of those.)
// The multiply-subtract below does not round a score as the maximum was, so a large score's rounding comes off the threshold: P
// stays within f16 for scores up to 2^27, and is cut to its end beyond.  (Scores rounded alike where they are that large: 371 us.)
constexpr float kWeightBits = 8.f, kRescaleThreshold = 7.9f, kScoreRounding = 0x1p-23f;
enum Bar {
  Q_FULL, K_FULL0, K_FULL1, RAW_FULL0, RAW_FULL1, RAW_FREE0, RAW_FREE1, V_FULL0, V_FULL1, QK_DONE0, QK_DONE1, PV_DONE0, PV_DONE1,
  P_FULL0, P_FULL1, ITEM_FULL0, ITEM_FULL1, ITEM_FREE0, ITEM_FREE1, O_FREE, EPI_FULL0, EPI_FULL1,
  INFO0, INFO1, INFO2, INFO3, FACTOR0, FACTOR1, ROWS_FULL, DRAIN, NUM_BARS
};
static_assert(NUM_BARS <= 32, "a barrier per lane");

template <int D_>
struct Geo {
  static constexpr int D = D_;
  static constexpr int Q_PART = BM * D, Q_BYTES = 2 * Q_PART;      // high and low e4m3 parts
  static constexpr int K_BYTES = BN * D;                           // codes
  static constexpr int V_SUB = BN * 128, V_BYTES = D / 64 * V_SUB;  // f16, 64 columns to a sub-tile
  static constexpr int OFF_Q = 0, OFF_K = OFF_Q + Q_BYTES, OFF_RAW = OFF_K + KST * K_BYTES, OFF_V = OFF_RAW + KST * K_BYTES;
  static constexpr int OFF_STAGE = OFF_V + KST * V_BYTES;          // 4 warps x 32 rows x 64 B of output
  // query rows as they are: D = 128 where their parts go (there is no room), D = 64 in a place of their own
  static constexpr int OFF_ROWS = D == 128 ? OFF_Q : OFF_STAGE + 4 * 2048;
  static constexpr int OFF_CTRL = OFF_STAGE + 4 * 2048 + (D == 128 ? 0 : BM * 128);  // barriers
  static constexpr int OFF_SLOTS = OFF_CTRL + 256;                 // two item descriptors of 8 ints
  static constexpr int OFF_MISC = OFF_SLOTS + 64;                  // TMEM address, abort flag
  static constexpr int OFF_TILES = OFF_MISC + 64;                  // 4 tiles: see Fp8Tile
  static constexpr int OFF_ROW = OFF_TILES + 256;                  // 2 items x 128 rows: the query row's power of two
  static constexpr int OFF_INV = OFF_ROW + 2 * 128 * 4;            // 2 items x 128 rows: 1 / row sum
  static constexpr int SMEM = OFF_INV + 2 * 128 * 4 + 1024;
  static constexpr int SBO = D == 128 ? 1024 : 512;                // eight rows of codes
  static constexpr int OCH = D / 32;
  static_assert(2 * (SMEM + 1024) <= 228 * 1024, "two blocks to an SM");
};
}  // namespace f8

struct PrefillFp8Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  __nv_bfloat16* out;
  int64_t out_stride;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int batch, hq, hkv, g;
  int pack, tile_tokens, inv_pack;  // query heads in a tile, its tokens, 2^16 / heads
  float scale_log2e;
  int64_t num_blocks;
  int* status;
  // few items: their keys in parts, a block to each (item * parts + part)
  int parts, items;
  int4* ws_items;  // [items]: first token, head, rows (0: nothing to sum up), parts
  float2* ws_ml;   // [blocks][128]: running maximum in log2 units, sum
  float4* ws_o;    // [blocks][D / 4][128]
};

// Shared-memory descriptor of e4m3 rows as TMA leaves them: 128-byte rows under the 128-byte swizzle, or 64 under the 64-byte one.
template <int D>
__device__ __forceinline__ uint64_t codes_desc(uint32_t smem_addr) {
  uint64_t d = static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(f8::Geo<D>::SBO >> 4) << 32;
  d |= 1ull << 46;
  d |= (D == 128 ? 2ull : 4ull) << 61;
  return d;
}
// Byte of 16-byte piece c of row r in such a tile.
template <int D>
__device__ __forceinline__ uint32_t code_piece(int r, int c) {
  return D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ (r >> 1 & 3)) << 4);
}
__device__ __forceinline__ void umma_f8_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// e4m3 x e4m3 -> fp32, both K-major; f16 x f16 -> fp32, B MN-major.
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) { return idesc_f8(m, n) | (1u << 16); }

// A tile's scales: K's; V's over the unit, as f16 pairs; what O is multiplied by (where the unit changes); the unit.
struct __align__(16) Fp8Tile {
  float k[4];
  uint32_t v[4];
  float change, unit, pad[2];
};
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

struct Fp8Item {
  int b, h, m0, q0, Lq, Lk, n_kv;  // n_kv key tiles, < 0: no more work
  int first;                       // of a part of an item's keys: its first tile
};

// Key tiles that the first `tokens` query tokens of a sequence see.
__device__ __forceinline__ int fp8_key_tiles(int tokens, int Lq, int Lk) {
  const int end = min(Lk, min(tokens, Lq) + (Lk - Lq));
  return end > 0 ? (end + f8::BN - 1) / f8::BN : 0;
}
// Query tiles of a sequence that see more than x key tiles (they are its last ones).
__device__ __forceinline__ int fp8_tiles_above(int x, int Lq, int Lk, int bmt) {
  const int tiles = (Lq + bmt - 1) / bmt, off = Lk - Lq;
  if (Lq <= 0 || Lk <= x * f8::BN) return 0;  // the last one sees the most
  // tile m sees more than x where off + (m + 1) bmt > 64 x
  const int least = x * f8::BN - off;  // tokens that see no more
  return least < 0 ? tiles : tiles - min(tiles - 1, least / bmt);
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(f8::NTHREADS, 2)
prefill_fp8_kernel(const PrefillFp8Params p, const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                   const __grid_constant__ CUtensorMap tmap_v) {
  using namespace f8;
  using G = Geo<D>;
  constexpr unsigned ALL = 0xffffffffu;
  extern __shared__ unsigned char smem_raw[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* base_ptr = smem_raw + (base - smem_u32(smem_raw));
  auto bar = [&](int i) { return base + G::OFF_CTRL + 8u * i; };
  volatile int* slots = reinterpret_cast<volatile int*>(base_ptr + G::OFF_SLOTS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base_ptr + G::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(base_ptr + G::OFF_MISC + 8);
  volatile int* parts_of_item = reinterpret_cast<volatile int*>(base_ptr + G::OFF_MISC + 16);  // SPLIT: whose part this block has
  float* row_factor = reinterpret_cast<float*>(base_ptr + G::OFF_ROW);
  float* inv_buf = reinterpret_cast<float*>(base_ptr + G::OFF_INV);
  float* unit_buf = reinterpret_cast<float*>(base_ptr + G::OFF_MISC + 24);  // 2 items: what O is held in at its end
  const int pack = p.pack, BMT = p.tile_tokens;
  auto token_of = [&](int row) { return row * p.inv_pack >> 16; };  // row / pack, row < 128

  pdl_trigger();
  if (warp == 9 && lane < NUM_BARS) {
    // by the four warps of a group: query rows, V, P, normalisers, O; an item slot is free when the softmax (4), the row (4)
    // warps, the MMA issuer and the two producers are done with it
    const bool by_four = lane == Q_FULL || lane == RAW_FREE0 || lane == RAW_FREE1 || lane == V_FULL0 || lane == V_FULL1 || lane == P_FULL0 ||
                         lane == P_FULL1 || lane == O_FREE || lane == EPI_FULL0 || lane == EPI_FULL1 || lane == FACTOR0 || lane == FACTOR1;
    mbar_init(bar(lane), by_four ? 4u : lane == ITEM_FREE0 || lane == ITEM_FREE1 ? 11u : 1u);
    if (lane == 0) {
      *abort_flag = 0;
      prefetch_tmap(&tmap_q);
      prefetch_tmap(&tmap_k);
      prefetch_tmap(&tmap_v);
    }
    mbar_fence_init();
  }
  if (warp == 10) tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
  pdl_wait();
  auto lens = [&](int b) { return make_int2(p.cu_q[b + 1] - p.cu_q[b], p.cu_k[b + 1] - p.cu_k[b]); };  // Lq, Lk
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + TMEM_O;
  auto tmem_s = [&](int st) { return tmem + st * 64; };

  auto tile_of = [&](int t) { return reinterpret_cast<const Fp8Tile*>(base_ptr + G::OFF_TILES + (t & 3) * sizeof(Fp8Tile)); };
  auto read_item = [&](int it) {
    volatile int* s = slots + (it & 1) * 8;
    Fp8Item x;
    x.b = s[0]; x.h = s[1]; x.m0 = s[2]; x.q0 = s[3];
    x.Lq = s[4]; x.Lk = s[5]; x.n_kv = s[6];
    x.first = SPLIT ? s[7] : 0;
    return x;
  };
  auto block_of = [&](const Fp8Item& x, int j) -> int64_t {  // of key tile j
    const int i = j * BN / kBlockSize;
    const int64_t blk = i < p.max_blocks ? p.block_tables[x.b * p.bt_stride + i] : -1;
    if (blk >= 0 && blk < p.num_blocks) return blk;
    if (lane == 0) atomicOr(p.status, NVLLM_STATUS_BAD_BLOCK);
    return 0;
  };

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHER));
    if (warp == 8) {
      // ---------------------------------------------------------------- TMA of the query rows and K; the scales
      const int g = lane & 3;
      int T = 0, loaded = 0, rows_loaded = 0;
      float most_unit = 0.f, unit = 0.f;
      bool ok = true;
#pragma unroll 1
      for (int it = 0; ok; ++it) {
        ok = __all_sync(ALL, wait_or_abort(bar(ITEM_FULL0 + (it & 1)), (it >> 1) & 1, abort_flag));
        if (!ok) break;
        const Fp8Item x = read_item(it);
        if (x.n_kv < 0) break;
        const int kvh = x.h / p.g;
        int64_t blk = block_of(x, x.first);
        auto scale_at = [&](int j) { return (blk * p.hkv + kvh) * kGroups + j * BN % kBlockSize / kScaleGroup + g; };
        float k = p.k_scale[scale_at(x.first)], v = p.v_scale[scale_at(x.first)];  // of tile j, group g
#pragma unroll 1
        for (int j = 0; j < x.n_kv; ++j) {
          const int t = T + j, st = t & 1, use = t >> 1, tile_no = x.first + j;
          const int row = static_cast<int>(blk * kBlockSize + tile_no * BN % kBlockSize);
          float k_next = 0.f, v_next = 0.f;
          if (j + 1 < x.n_kv) {
            if ((tile_no + 1) % (kBlockSize / BN) == 0) blk = block_of(x, tile_no + 1);
            k_next = p.k_scale[scale_at(tile_no + 1)], v_next = p.v_scale[scale_at(tile_no + 1)];
          }
          ok = __all_sync(ALL, use == 0 || wait_or_abort(bar(QK_DONE0 + st), (use - 1) & 1, abort_flag));
          if (!ok) break;
          // K's stage is free, and so is the record of tile t - 4: the scores of tile t - 2 were issued behind that tile's product,
          // so behind its softmax and its V.  Nobody may read a record after he has reported his part of its tile.
          if (lane == 0) {
            mbar_expect_tx(bar(K_FULL0 + st), G::K_BYTES);
            tma_load_3d(base + G::OFF_K + st * G::K_BYTES, &tmap_k, bar(K_FULL0 + st), 0, kvh, row);
          }
          ++loaded;
          if (tile_no * BN + g * kScaleGroup >= x.Lk) k = 1.f, v = 0.f;  // a group behind the end may hold anything
          float most = fmaxf(v, __shfl_xor_sync(ALL, v, 1));
          most = fmaxf(most, __shfl_xor_sync(ALL, most, 2));
          const float before = unit;
          if (j == 0) unit = most, most_unit = 0.f;
          else if (most > unit * 128.f || (most > 0.f && most * 0x1p14f < unit)) unit = fmaxf(most, most_unit * 0x1p-60f);
          unit = fminf(fmaxf(unit, 0x1p-126f), kLargestUnit);
          most_unit = fmaxf(most_unit, unit);
          Fp8Tile& tile = *reinterpret_cast<Fp8Tile*>(base_ptr + G::OFF_TILES + (t & 3) * sizeof(Fp8Tile));
          if (lane < 4) {
            const float ratio = mul_subnormal(v, 1.f / unit);
            tile.k[g] = k;
            asm("cvt.rn.f16x2.f32 %0, %1, %1;" : "=r"(tile.v[g]) : "f"(ratio));
            if (g == 0) {
              tile.change = j > 0 && unit != before ? before / unit : 1.f;
              tile.unit = unit;
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(INFO0 + (t & 3)));
          k = k_next, v = v_next;
          if (j == 0) {
            // The query rows, as they are: their place is free once the previous item's last scores are there, or, in a place of
            // their own, once its rows have been taken.
            if constexpr (D == 128) ok = __all_sync(ALL, t == 0 || wait_or_abort(bar(QK_DONE0 + ((t - 1) & 1)), ((t - 1) >> 1) & 1, abort_flag));
            else ok = __all_sync(ALL, it == 0 || wait_or_abort(bar(FACTOR0 + ((it - 1) & 1)), ((it - 1) >> 1) & 1, abort_flag));
            if (!ok) break;
            if (lane == 0) {
              mbar_expect_tx(bar(ROWS_FULL), D / 64 * pack * BMT * 128);
              tma_load_3d(base + G::OFF_ROWS, &tmap_q, bar(ROWS_FULL), 0, x.h, x.q0 + x.m0);
              if constexpr (D == 128) tma_load_3d(base + G::OFF_ROWS + BM * 128, &tmap_q, bar(ROWS_FULL), 64, x.h, x.q0 + x.m0);
            }
            ++rows_loaded;
          }
        }
        if (!ok) break;
        T += x.n_kv;
        if (lane == 0) mbar_arrive(bar(ITEM_FREE0 + (it & 1)));
      }
      // no copy is in flight when the block ends, whoever gave up
#pragma unroll 1
      for (int t = max(loaded - 2, 0); t < loaded; ++t) (void)mbar_wait(bar(K_FULL0 + (t & 1)), (t >> 1) & 1);
      if (rows_loaded > 0) (void)mbar_wait(bar(ROWS_FULL), (rows_loaded - 1) & 1);
    } else if (warp == 10) {
      // ---------------------------------------------------------------- TMA of V
      if (elect_one()) {
        int T = 0, loaded = 0;
        bool ok = true;
#pragma unroll 1
        for (int it = 0; ok; ++it) {
          if (!(ok = wait_or_abort(bar(ITEM_FULL0 + (it & 1)), (it >> 1) & 1, abort_flag))) break;
          const Fp8Item x = read_item(it);
          if (x.n_kv < 0) break;
          const int kvh = x.h / p.g;
          int64_t blk = 0;
#pragma unroll 1
          for (int j = 0; j < x.n_kv; ++j) {
            const int t = T + j, st = t & 1, use = t >> 1, tile_no = x.first + j;
            if (j == 0 || tile_no % (kBlockSize / BN) == 0) blk = block_of(x, tile_no);
            if (use > 0 && !(ok = wait_or_abort(bar(RAW_FREE0 + st), (use - 1) & 1, abort_flag))) break;
            mbar_expect_tx(bar(RAW_FULL0 + st), G::K_BYTES);
            tma_load_3d(base + G::OFF_RAW + st * G::K_BYTES, &tmap_v, bar(RAW_FULL0 + st), 0, kvh,
                        static_cast<int>(blk * kBlockSize + tile_no * BN % kBlockSize));
            ++loaded;
          }
          if (!ok) break;
          T += x.n_kv;
          mbar_arrive(bar(ITEM_FREE0 + (it & 1)));
        }
#pragma unroll 1
        for (int t = max(loaded - 2, 0); t < loaded; ++t) (void)mbar_wait(bar(RAW_FULL0 + (t & 1)), (t >> 1) & 1);
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------------- MMA issuer
      if (elect_one()) {
        constexpr uint32_t idesc_qk = idesc_f8(BM, BN), idesc_pv = idesc_f16(BM, D);
        const uint64_t q_desc = codes_desc<D>(base + G::OFF_Q), k_desc = codes_desc<D>(base + G::OFF_K);
        const uint64_t v_desc = umma_desc(base + G::OFF_V, G::V_SUB, 1024);
        auto issue_qk = [&](int t) -> bool {
          const int st = t & 1;
          if (!wait_or_abort(bar(K_FULL0 + st), (t >> 1) & 1, abort_flag)) return false;
          tc_fence_after();
          const uint64_t kd = k_desc + static_cast<uint64_t>(st * (G::K_BYTES >> 4));
#pragma unroll
          for (int part = 0; part < 2; ++part)
#pragma unroll
            for (int ks = 0; ks < D / 32; ++ks)
              umma_f8_ss(tmem_s(st), q_desc + ((part * G::Q_PART + ks * 32) >> 4), kd + ((ks * 32) >> 4), idesc_qk, part > 0 || ks > 0);
          umma_commit(bar(QK_DONE0 + st));
          return true;
        };
        int T = 0;
        bool ok = true;
#pragma unroll 1
        for (int it = 0; ok; ++it) {
          if (!(ok = wait_or_abort(bar(ITEM_FULL0 + (it & 1)), (it >> 1) & 1, abort_flag))) break;
          const Fp8Item x = read_item(it);
          if (x.n_kv < 0) break;
          if (!(ok = wait_or_abort(bar(Q_FULL), it & 1, abort_flag))) break;
#pragma unroll 1
          for (int j = -1; j < x.n_kv; ++j) {
            const int t = T + j, st = t & 1, ph = (t >> 1) & 1;
            if (j + 1 < x.n_kv && !(ok = issue_qk(t + 1))) break;  // the next scores run under this tile's softmax
            if (j < 0) continue;
            if (!(ok = wait_or_abort(bar(V_FULL0 + st), ph, abort_flag))) break;
            if (!(ok = wait_or_abort(bar(P_FULL0 + st), ph, abort_flag))) break;
            // the first product of an item overwrites O: the previous item's must have been read
            if (j == 0 && it > 0 && !(ok = wait_or_abort(bar(O_FREE), (it - 1) & 1, abort_flag))) break;
            tc_fence_after();
            const uint64_t vd = v_desc + static_cast<uint64_t>(st * (G::V_BYTES >> 4));
#pragma unroll
            for (int ks = 0; ks < BN / 16; ++ks)
              umma_ts(tmem_o, tmem_s(st) + ks * 8, vd + static_cast<uint64_t>((ks * 2048) >> 4), idesc_pv, (j > 0 || ks > 0) ? 1u : 0u);
            umma_commit(bar(PV_DONE0 + st));
          }
          if (!ok) break;
          T += x.n_kv;
          mbar_arrive(bar(ITEM_FREE0 + (it & 1)));
        }
        if (!ok) {  // make sure nothing is still running on TMEM before it is freed
          umma_commit(bar(DRAIN));
          (void)mbar_wait(bar(DRAIN), 0);
        }
      }
    } else {
      // ---------------------------------------------------------------- items, one ahead of the others; rows that see no key
      const int hgroups = p.hq / pack;
      // Query tiles of all sequences that see more than x key tiles.
      const int2 mine = lane < p.batch ? lens(lane) : make_int2(0, 0);
      auto length = [&](int b) { return b == lane ? mine : lens(b); };
      auto above = [&](int x) {
        int n = fp8_tiles_above(x, mine.x, mine.y, BMT);
#pragma unroll 1
        for (int b = lane + 32; b < p.batch; b += 32) {
          const int2 len = lens(b);
          n += fp8_tiles_above(x, len.x, len.y, BMT);
        }
        return __reduce_add_sync(ALL, static_cast<unsigned>(n));
      };
      int longest = 0;
#pragma unroll 1
      for (int b = lane; b < p.batch; b += 32) longest = max(longest, length(b).y);
      longest = (__reduce_max_sync(ALL, longest) + BN - 1) / BN;
      const unsigned total = above(0) * hgroups;  // items; tiles that see no key are none
      bool ok = true;
#pragma unroll 1
      for (int it = 0;; ++it) {
        const unsigned drawn = SPLIT ? (it == 0 ? blockIdx.x / p.parts : total)
                                     : it * gridDim.x + (it & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        Fp8Item x{};
        x.n_kv = -1;
        if (drawn < total) {
          const unsigned rank = drawn / hgroups;
          x.h = (drawn - rank * hgroups) * pack;
          int lo = 1, hi = longest;  // its key tiles: the least n with above(n) <= rank (above(longest) = 0)
#pragma unroll 1
          while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (above(mid) <= rank) hi = mid;
            else lo = mid + 1;
          }
          x.n_kv = lo;
          unsigned k = rank - above(lo);  // its number among the tiles with as many
#pragma unroll 1
          for (int b0 = 0; b0 < p.batch; b0 += 32) {
            const int b = b0 + lane;
            unsigned n = 0;
            if (b < p.batch) {
              const int2 len = length(b);
              n = fp8_tiles_above(lo - 1, len.x, len.y, BMT) - fp8_tiles_above(lo, len.x, len.y, BMT);
            }
            unsigned incl = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
              const unsigned v = __shfl_up_sync(ALL, incl, d);
              if (lane >= d) incl += v;
            }
            const unsigned hit = __ballot_sync(ALL, incl > k);
            if (hit) {
              const int src = __ffs(hit) - 1;
              x.b = b0 + src;
              k -= __shfl_sync(ALL, incl - n, src);
              break;
            }
            k -= __shfl_sync(ALL, incl, 31);
          }
          x.Lq = lens(x.b).x;
          x.Lk = lens(x.b).y;
          x.q0 = p.cu_q[x.b];
          x.m0 = ((x.Lq + BMT - 1) / BMT - 1 - fp8_tiles_above(lo, x.Lq, x.Lk, BMT) - static_cast<int>(k)) * BMT;
        }
        if (SPLIT && x.n_kv > 0) {
          const int parts = max(1, min(p.parts, x.n_kv / 2)), part = blockIdx.x % p.parts;
          x.first = static_cast<int>(static_cast<int64_t>(x.n_kv) * part / parts);
          x.n_kv = part < parts ? static_cast<int>(static_cast<int64_t>(x.n_kv) * (part + 1) / parts) - x.first : -1;
          if (lane == 0) {
            *parts_of_item = parts;
            if (part == 0) p.ws_items[drawn] = make_int4(x.q0 + x.m0, x.h, parts > 1 ? min(BMT, x.Lq - x.m0) * pack : 0, parts);
          }
        } else if (SPLIT && lane == 0 && it == 0 && blockIdx.x % p.parts == 0) {
          p.ws_items[drawn] = make_int4(0, 0, 0, 0);  // no such item
        }
        if (it >= 2) ok = wait_or_abort(bar(ITEM_FREE0 + (it & 1)), ((it >> 1) - 1) & 1, abort_flag);
        if (!__all_sync(ALL, ok)) break;
        if (lane == 0) {
          volatile int* s = slots + (it & 1) * 8;
          s[0] = x.b; s[1] = x.h; s[2] = x.m0; s[3] = x.q0;
          s[4] = x.Lq; s[5] = x.Lk; s[6] = x.n_kv;
          if (SPLIT) s[7] = x.first;
          mbar_arrive(bar(ITEM_FULL0 + (it & 1)));
          if (x.n_kv > 0) {  // its query rows are on the path from the item before: to L2
            tma_prefetch_3d(&tmap_q, 0, x.h, x.q0 + x.m0);
            if constexpr (D == 128) tma_prefetch_3d(&tmap_q, 64, x.h, x.q0 + x.m0);
          }
        }
        __syncwarp();
        if (x.n_kv < 0) break;
      }
#pragma unroll 1
      for (int b = blockIdx.x; b < p.batch; b += gridDim.x) {
        const int Lq = lens(b).x, Lk = lens(b).y, dead = Lk <= 0 ? Lq : Lk < Lq ? (Lq - Lk) / BMT * BMT : 0;
        const int per_row = p.hq * (D / 8);
        const int64_t q0 = p.cu_q[b];
#pragma unroll 1
        for (int t = 0; t < dead; ++t)
#pragma unroll 1
          for (int i = lane; i < per_row; i += 32)
            reinterpret_cast<uint4*>(p.out + (q0 + t) * p.out_stride)[i] = make_uint4(0, 0, 0, 0);
      }
    }
  } else if (warp < 4) {
    // ------------------------------------------------------------------ softmax rows
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    const int r = warp * 32 + lane;
    const int r_tok = token_of(r);
    const uint32_t lane_addr = static_cast<uint32_t>(warp * 32) << 16;
    int T = 0;
    bool ok = true;
#pragma unroll 1
    for (int it = 0; ok; ++it) {
      if (!(ok = wait_or_abort(bar(ITEM_FULL0 + (it & 1)), (it >> 1) & 1, abort_flag))) break;
      const Fp8Item x = read_item(it);
      if (x.n_kv < 0) break;
      if (!(ok = wait_or_abort(bar(FACTOR0 + (it & 1)), (it >> 1) & 1, abort_flag))) break;
      const float factor = row_factor[(it & 1) * 128 + r];
      const int qi = x.m0 + r_tok, off = x.Lk - x.Lq;
      float m_used = -INFINITY, l = 0.f, unit = 0.f;
#pragma unroll 1
      for (int j = 0; j < x.n_kv; ++j) {
        const int t = T + j, st = t & 1, ph = (t >> 1) & 1;
        const uint32_t scores = tmem_s(st) + lane_addr;
        if (!(ok = wait_or_abort(bar(QK_DONE0 + st), ph, abort_flag))) break;
        tc_fence_after();
        uint32_t s[64];
        tmem_ld32(scores, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld32(scores + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        if (!(ok = wait_or_abort(bar(INFO0 + (t & 3)), (t >> 2) & 1, abort_flag))) break;
        const Fp8Tile& tile = *tile_of(t);
        float ks[4];
        *reinterpret_cast<float4*>(ks) = *reinterpret_cast<const float4*>(tile.k);
        const float change = tile.change;
        unit = tile.unit;  // goes on with the rows' sums: the record is the next tiles' once P is reported
#pragma unroll
        for (int g = 0; g < 4; ++g) ks[g] = fmaxf(ks[g] * factor, 0x1p-126f);  // not zero, which -inf of a masked score must not meet
        const int j0 = (x.first + j) * BN;
        tmem_wait_ld();
        if ((j0 + BN - 1 > x.m0 + off) || (j0 + BN > x.Lk)) {  // tile touches the diagonal or the end
          const int limit = min(qi + off, x.Lk - 1) - j0;        // columns c <= limit are visible
#pragma unroll
          for (int c = 0; c < 64; ++c)
            if (c > limit) s[c] = 0xff800000u;  // -inf
        }
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int c = g * 16; c < g * 16 + 16; c += 4) {
            m2[0] = fmax3(m2[0], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
            m2[1] = fmax3(m2[1], __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
          }
          mx = fmaxf(mx, fmaxf(m2[0], m2[1]) * ks[g]);
        }
        const float m_new = fmaxf(m_used, mx);
        // lazy rescale: the old reference maxima stay until one of the warp has been outgrown by the threshold; then all follow
        if (change != 1.f || __any_sync(ALL, m_new - m_used > fmaf(fabsf(m_new), -kScoreRounding, kRescaleThreshold))) {
          float alpha = 1.f;
          if (m_new > m_used) {
            alpha = (m_used == -INFINITY) ? 0.f : fast_exp2(m_used - m_new);
            m_used = m_new;
            l *= alpha;
          }
          alpha *= change;
          if (j > 0) {  // O holds tiles 0..j-1 of this item once the previous product has finished
            if (!(ok = wait_or_abort(bar(PV_DONE0 + ((t - 1) & 1)), ((t - 1) >> 1) & 1, abort_flag))) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < G::OCH; ++c) {
              uint32_t o[32];
              tmem_ld32(tmem_o + lane_addr + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st32(tmem_o + lane_addr + c * 32, o);
            }
          }
        }
        const float msub = (m_used == -INFINITY) ? 0.f : m_used - kWeightBits;
        // p = 2^(s * scale - m + 8), and so are l and O: the multiply-subtract and the row sum run two lanes at a time
        const uint64_t nmsub2 = pack2(-msub, -msub);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint64_t scale2 = pack2(ks[g], ks[g]);
#pragma unroll
          for (int c = g * 8; c < g * 8 + 8; ++c) {  // P is packed in place: s[c] <- (p[2c], p[2c+1])
            float a0, a1;
            unpack2(fma2(pack2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), scale2, nmsub2), a0, a1);
            const float p0 = fast_exp2(a0), p1 = fast_exp2(a1);
            sum2[c & 1] = add2(sum2[c & 1], pack2(p0, p1));
            asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(s[c]) : "f"(p1), "f"(p0));
          }
        }
        {
          float t0, t1, t2, t3;
          unpack2(sum2[0], t0, t1);
          unpack2(sum2[1], t2, t3);
          l += (t0 + t1) + (t2 + t3);
        }
        tmem_st32(scores, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL0 + st));
      }
      if (!ok) break;
      T += x.n_kv;
      // what takes O to the result, or to its part of it, goes to the row warps; no key: zeros; a sum that is NaN stays one
      float by = l > 0.f ? 1.f / l : l;
      if (SPLIT && *parts_of_item > 1) {
        by = 1.f / (1 << static_cast<int>(kWeightBits));  // sums of large values end where fp32 does as it is
        p.ws_ml[static_cast<int64_t>(blockIdx.x) * BM + r] = make_float2(m_used, l * by);
      }
      inv_buf[(it & 1) * 128 + r] = by;
      if (r == 0) unit_buf[it & 1] = unit;
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(EPI_FULL0 + (it & 1)));
        mbar_arrive(bar(ITEM_FREE0 + (it & 1)));
      }
    }
  } else {
    // ------------------------------------------------------------------ query rows in, V to f16, results out
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_ROWS));
    const int ew = warp - 4, r = ew * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(ew * 32) << 16;
    unsigned char* stage = base_ptr + G::OFF_STAGE + ew * 2048;
    // Thread = query row: its power of two, then its two parts, eight values at a time (f16 holds them: 128 <= max < 256): the
    // nearest codes, and the nearest ones of what is left.  Run once an item, so short: code that is not in the instruction
    // cache comes at 25 cycles an instruction (unrolled, this took 8000 cycles).
    // D = 128: TMA has brought the bf16 values into the place of the parts, in two sub-tiles of 64 columns, rows of 128 bytes as
    // the parts have; a thread stays within its own rows' bytes and writes none before what lies there has been read: pieces
    // 0 to 7, then 15 down to 8, the first half's low parts by way of this thread's 64 bytes of the patch for results.
    auto take_rows = [&](const Fp8Item& x, int it, int last) {  // last: the last tile of the item before
      if (!wait_or_abort(bar(ROWS_FULL), it & 1, abort_flag)) return false;
      const bool live = token_of(r) < BMT;  // rows behind a sequence's end hold something that nobody looks at
      const uint32_t from = base + G::OFF_ROWS + r * 128 + ((r & 7) << 4);  // piece i, eight values: the sub-tile's, ^ i * 16
      auto piece = [&](int i) { return ld_shared16((from + (i >> 3) * (BM * 128)) ^ ((i & 7) << 4)); };
      uint32_t m = 0;  // the largest magnitudes, two columns at a time; infinities and NaN stay what they are
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        const uint4 a = piece(i);
        m = max_magnitude(max_magnitude(a.x, a.y), max_magnitude(max_magnitude(a.z, a.w), m));
      }
      m &= 0x7fff7fffu;
      m = live ? max(m & 0xffffu, m >> 16) : 0;
      const uint32_t spoilt = m >= 0x7f80u ? 0x7fu : 0u;  // an infinity or NaN: so is the row, by its first code
      const int e = min(max(static_cast<int>(m >> 7), 20), 254) - 127;  // 2^e <= max |q| < 2^(e + 1)
      const float f = power_of_two(7 - e);
      row_factor[(it & 1) * 128 + r] = p.scale_log2e * power_of_two(e - 7);
      if (D == 64 && it > 0 && !wait_or_abort(bar(QK_DONE0 + (last & 1)), (last >> 1) & 1, abort_flag)) return false;
      // pieces of the parts, two of these to one: the high part's row and swizzle, the low part's, the patch's
      const uint32_t to_high = base + G::OFF_Q + code_piece<D>(r, 0), to_low = to_high + G::Q_PART;
      const uint32_t to_aside = smem_u32(stage) + lane * 64 + ((lane >> 1 & 3) << 4);
#pragma unroll 1
      for (int n = 0; n < D / 8; ++n) {
        const int i = n < 8 ? n : 23 - n;
        const uint4 a = piece(i);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w}, at = (i >> 1) << 4, half = (i & 1) * 8;
        uint32_t h[4], l[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t y, rest;
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(__uint_as_float(w[k] & 0xffff0000u) * f), "f"(__uint_as_float(w[k] << 16) * f));
          h[k] = e4m3x2_of_f16x2(y);
          asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(rest) : "r"(y), "r"(f16x2_of_low(h[k])));
          l[k] = e4m3x2_of_f16x2(rest);
        }
        if (n == 0) h[0] |= spoilt;
        st_shared8((to_high ^ at) + half, make_uint2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[2], h[3], 0x5410)));
        st_shared8((D == 128 && n < 8 ? to_aside ^ at : to_low ^ at) + half, make_uint2(__byte_perm(l[0], l[1], 0x5410), __byte_perm(l[2], l[3], 0x5410)));
      }
      if constexpr (D == 128) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) st_shared16(to_low ^ c << 4, ld_shared16(to_aside ^ c << 4));
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(Q_FULL));
        mbar_arrive(bar(FACTOR0 + (it & 1)));
      }
      return true;
    };
    // Tile t (the j-th of item x) of V: 16 codes at a time to two 16-byte pieces of f16, times the group's scale over the unit.
    // Eight lanes take two rows' halves whose pieces are in different banks both where they come from and where they go: at
    // D = 64 neighbouring rows, at D = 128 rows whose numbers differ by the bits of 5.  The next of a thread's pieces lie 16
    // (D = 128) or 32 rows on, so in places a constant apart.
    constexpr int STEPS = D / 32, STEP_ROWS = BN / STEPS;  // pieces of a thread
    const int v_row = D == 64 ? r >> 2 : (r >> 6) * 8 + ((r >> 4 & 3) ^ (r & 4 ? 5 : 0)), v_piece = D == 64 ? r & 3 : (r & 3) | (r & 8) >> 1;
    const unsigned char* v_from = base_ptr + G::OFF_RAW + code_piece<D>(v_row, v_piece);
    unsigned char* v_to = base_ptr + G::OFF_V + (v_piece >> 2) * G::V_SUB + v_row * 128 + (((v_piece & 3) * 2 ^ (v_row & 7)) << 4);
    auto convert = [&](const Fp8Item& x, int j, int t) {
      const int st = t & 1, use = t >> 1, rows = x.Lk - (x.first + j) * BN;
      if (!wait_or_abort(bar(INFO0 + (t & 3)), (t >> 2) & 1, abort_flag)) return false;
      uint32_t by[4];
      *reinterpret_cast<uint4*>(by) = *reinterpret_cast<const uint4*>(tile_of(t)->v);
      if (!wait_or_abort(bar(RAW_FULL0 + st), use & 1, abort_flag)) return false;
      if (use > 0 && !wait_or_abort(bar(PV_DONE0 + st), (use - 1) & 1, abort_flag)) return false;
      uint4 code[STEPS];
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        code[i] = *reinterpret_cast<const uint4*>(v_from + st * G::K_BYTES + i * (STEP_ROWS * D));
      if (rows < BN) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
          if (i * STEP_ROWS + v_row >= rows) code[i] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const uint32_t f = D == 128 ? by[i] : r < 64 ? by[2 * i] : by[2 * i + 1];  // of rows 16 i .. or 32 i ..: their groups
        unsigned char* to = v_to + st * G::V_BYTES + i * (STEP_ROWS * 128);
        *reinterpret_cast<uint4*>(to) = make_uint4(
            mul_f16x2(f16x2_of_low(code[i].x), f), mul_f16x2(f16x2_of_high(code[i].x), f), mul_f16x2(f16x2_of_low(code[i].y), f), mul_f16x2(f16x2_of_high(code[i].y), f));
        to = reinterpret_cast<unsigned char*>(reinterpret_cast<uintptr_t>(to) ^ 16);  // the odd neighbour: pieces 2 c and 2 c + 1
        *reinterpret_cast<uint4*>(to) = make_uint4(
            mul_f16x2(f16x2_of_low(code[i].z), f), mul_f16x2(f16x2_of_high(code[i].z), f), mul_f16x2(f16x2_of_low(code[i].w), f), mul_f16x2(f16x2_of_high(code[i].w), f));
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(V_FULL0 + st));
        mbar_arrive(bar(RAW_FREE0 + st));
      }
      return true;
    };
    // A part of an item's keys: O in 32 bits goes to the workspace, four columns of all rows side by side.
    auto set_aside = [&](const Fp8Item& x, float by, float unit) {
      const int rows = min(BMT, x.Lq - x.m0) * pack;
      float4* mine = p.ws_o + static_cast<int64_t>(blockIdx.x) * (D / 4) * BM + r;
#pragma unroll 1
      for (int c = 0; c < G::OCH; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem_o + lane_addr + c * 32, o);
        tmem_wait_ld();
        if (r < rows) {
#pragma unroll
          for (int k = 0; k < 32; k += 4)
            mine[(c * 8 + k / 4) * BM] = make_float4(__uint_as_float(o[k]) * by * unit, __uint_as_float(o[k + 1]) * by * unit,
                                                     __uint_as_float(o[k + 2]) * by * unit, __uint_as_float(o[k + 3]) * by * unit);
        }
      }
      return true;
    };
    // Results of item number `done`, whose last tile was `last`.  Its record may be another tile's by now: what is needed of it came
    // with the row's sum.
    auto results = [&](const Fp8Item& x, int done, int last) {
      if (!wait_or_abort(bar(EPI_FULL0 + (done & 1)), (done >> 1) & 1, abort_flag)) return false;
      const float inv = inv_buf[(done & 1) * 128 + r], unit = unit_buf[done & 1];  // one after the other: their product may be subnormal
      if (!wait_or_abort(bar(PV_DONE0 + (last & 1)), (last >> 1) & 1, abort_flag)) return false;
      tc_fence_after();
      if (SPLIT && *parts_of_item > 1) return set_aside(x, inv, unit);
      // O / l -> bf16, 32 columns at a time through this warp's patch of shared memory
      const int srow = lane >> 2, spiece = lane & 3;
      __nv_bfloat16* out_tile = p.out + static_cast<int64_t>(x.q0 + x.m0) * p.out_stride + x.h * D;
      const int toks_valid = min(BMT, x.Lq - x.m0);
#pragma unroll 1
      for (int c = 0; c < G::OCH; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem_o + lane_addr + c * 32, o);
        tmem_wait_ld();
        if (c == G::OCH - 1) {  // O is in registers: the next item's first product may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(O_FREE));
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint4 v;
          v.x = pack_bf16x2(__uint_as_float(o[8 * k]) * inv * unit, __uint_as_float(o[8 * k + 1]) * inv * unit);
          v.y = pack_bf16x2(__uint_as_float(o[8 * k + 2]) * inv * unit, __uint_as_float(o[8 * k + 3]) * inv * unit);
          v.z = pack_bf16x2(__uint_as_float(o[8 * k + 4]) * inv * unit, __uint_as_float(o[8 * k + 5]) * inv * unit);
          v.w = pack_bf16x2(__uint_as_float(o[8 * k + 6]) * inv * unit, __uint_as_float(o[8 * k + 7]) * inv * unit);
          *reinterpret_cast<uint4*>(stage + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)) = v;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int lr = i * 8 + srow, row = ew * 32 + lr;
          const int tok = token_of(row), hh = row - tok * pack;
          const uint4 v = *reinterpret_cast<const uint4*>(stage + lr * 64 + ((spiece ^ ((lr >> 1) & 3)) << 4));
          if (tok < toks_valid)
            *reinterpret_cast<uint4*>(out_tile + static_cast<int64_t>(tok) * p.out_stride + hh * D + c * 32 + spiece * 8) = v;
        }
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(bar(ITEM_FREE0 + (done & 1)));
      return true;
    };
    // An item's results are written when the next one's rows and first tile are there, whose products run meanwhile.
    Fp8Item before{};
    int T = 0;
    bool ok = true;
#pragma unroll 1
    for (int it = 0; ok; ++it) {
      if (!(ok = wait_or_abort(bar(ITEM_FULL0 + (it & 1)), (it >> 1) & 1, abort_flag))) break;
      const Fp8Item x = read_item(it);
      if (x.n_kv > 0 && !(ok = take_rows(x, it, T - 1))) break;
#pragma unroll 1
      for (int j = 0; ok && j < max(x.n_kv, 1); ++j) {
        if (x.n_kv > 0 && !(ok = convert(x, j, T + j))) break;
        if (j == 0 && it > 0) ok = results(before, it - 1, T - 1);
      }
      if (x.n_kv < 0) break;
      T += x.n_kv;
      before = x;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(p.status, NVLLM_STATUS_TIMEOUT);
  if (warp == 10) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// What an item's parts add up to: a thread has a row's four columns of all parts, `1 << log_rows` rows side by side.  It loads
// eight parts at a time, before it is known how many there are (the workspace holds as many for every item): one latency.
// (The block that reports an item's last part as the one that sums them up has only its own loads to hide the latency
// with: 20 us for 50 rows in 5 parts.)
template <int D>
__global__ void __launch_bounds__(256) prefill_fp8_join_kernel(const PrefillFp8Params p, int log_rows) {
  using namespace f8;
  const int t = blockIdx.x * 256 + threadIdx.x, row = t & ((1 << log_rows) - 1), c = (t >> log_rows) & (D / 4 - 1);
  const int item = (t >> log_rows) / (D / 4);
  pdl_prologue();
  if (item >= p.items) return;
  const int4 what = p.ws_items[item];
  const float2* ml = p.ws_ml + static_cast<int64_t>(item) * p.parts * BM + row;
  const float4* from = p.ws_o + (static_cast<int64_t>(item) * p.parts * (D / 4) + c) * BM + row;
  float top = -INFINITY, sum = 0.f;
  float4 acc{};
#pragma unroll 1
  for (int i0 = 0; i0 < p.parts; i0 += 8) {
    float2 s[8];
    float4 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i0 + i < p.parts) s[i] = ml[(i0 + i) * BM], o[i] = from[static_cast<int64_t>(i0 + i) * (D / 4) * BM];
    float high = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i0 + i >= what.w) s[i] = make_float2(-INFINITY, 0.f);
      high = fmaxf(high, s[i].x);
    }
    const float old = top == -INFINITY ? 0.f : fast_exp2(top - high);
    sum *= old, acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
    top = high;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float w = s[i].x == -INFINITY ? 0.f : fast_exp2(s[i].x - top);
      sum = fmaf(s[i].y, w, sum);  // no maximum but a sum: NaN, which zero times it stays
      if (s[i].x != -INFINITY) {
        acc.x = fmaf(o[i].x, w, acc.x), acc.y = fmaf(o[i].y, w, acc.y);
        acc.z = fmaf(o[i].z, w, acc.z), acc.w = fmaf(o[i].w, w, acc.w);
      }
    }
  }
  if (row >= what.z) return;
  const float by = sum > 0.f ? 1.f / sum : sum;  // no key: zeros; a sum that is NaN stays one
  const int tok = row * p.inv_pack >> 16, hh = row - tok * p.pack;
  *reinterpret_cast<uint2*>(p.out + static_cast<int64_t>(what.x + tok) * p.out_stride + (what.y + hh) * D + c * 4) =
      make_uint2(pack_bf16x2(acc.x * by, acc.y * by), pack_bf16x2(acc.z * by, acc.w * by));
}

// ---- host side ---------------------------------------------------------------------------

// Heads packed into a query tile: the largest divisor of the group size that is at most 8.
static int heads_in_tile(int g) {
  int pack = 1;
  for (int n = 2; n <= 8; ++n)
    if (g % n == 0) pack = n;
  return pack;
}

template <int D, bool SPLIT>
static int prepare_prefill_fp8() {
  cudaError_t e = cudaFuncSetAttribute(prefill_fp8_kernel<D, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, f8::Geo<D>::SMEM);
  // The warp groups trade registers inside the pool the block gets at launch: a build with fewer could never satisfy the
  // softmax group's request, and that request waits without a bound.
  cudaFuncAttributes attr;
  if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, prefill_fp8_kernel<D, SPLIT>);
  if (e != cudaSuccess) return fail(NVLLM_E_CUDA, "prefill_fp8: set-up failed: %s", cudaGetErrorString(e));
  if (attr.numRegs < f8::REGS_LAUNCH)
    return fail(NVLLM_E_CUDA, "prefill_fp8: built with %d registers per thread, the warp groups' hand-over needs %d", attr.numRegs,
                f8::REGS_LAUNCH);
  return NVLLM_OK;
}

// Items of a launch at most, as far as the host knows.
static int64_t prefill_fp8_items(int hq, int g, int max_seqlen_q, int batch) {
  const int pack = heads_in_tile(g), tokens = f8::BM / pack;
  return static_cast<int64_t>((max_seqlen_q + tokens - 1) / tokens) * (hq / pack) * batch;
}
// The parts that an item's keys go into; 1: whole items.  A tile takes a block 0.9 us, which is latency, a part more 0.1 us of
// summing up, and a split at all 2 to 4 us (one sequence, 16 heads over 8 of dim 128, 600 cached tokens and 25 new ones: whole
// 15.6, 5 parts 12.7, 24 parts 16.6 us; 16000 and 16: whole 191, 12 parts 35.5, 32 parts 26.8; 5000 and 1: 65.7, 12 parts 19.3,
// 32 parts 23.3; 700 new ones alone: whole 18.4, 3 parts 21.8; 400 and 300: whole 18.5, 2 parts 17.9).  So none where an item has
// fewer than 9 tiles, and about 2 sqrt(tiles) parts, two tiles to each at least, as many as there are blocks for.
static int prefill_fp8_parts(int64_t items, int max_seqlen_q, int max_seqlen_k, int blocks) {
  const int64_t tiles = (max_seqlen_k - max_seqlen_q / 2 + int64_t{f8::BN - 1}) / f8::BN;  // of an item in the middle of its queries
  if (tiles < 9) return 1;
  const int64_t most = std::min<int64_t>(tiles / 2, 32);
  int parts = 1;
  while (parts < most && (parts + 1) * items <= blocks && parts * parts < 4 * tiles) ++parts;
  return parts;
}
static int prefill_fp8_blocks() {
  const int sms = num_sms();
  return sms > 0 ? 2 * sms : 512;  // no device: as if there were more than any has
}
constexpr int64_t kFp8CounterArea = 16384 * 4;  // at the workspace's head, left as it is: the decode's, whose workspace this may be

template <int D>
static int launch_prefill_fp8(PrefillFp8Params& p, const void* k_cache, const void* v_cache, int64_t total_q, int max_seqlen_q,
                              int max_seqlen_k, void* workspace, cudaStream_t stream) {
  using G = f8::Geo<D>;
  static bool ready[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return fail(NVLLM_E_NO_DEVICE, "prefill_fp8: device index %d out of range", dev);
  if (!ready[dev]) {  // both: another's first launch may be captured
    int rc = prepare_prefill_fp8<D, false>();
    if (rc == NVLLM_OK) rc = prepare_prefill_fp8<D, true>();
    if (rc) return rc;
    ready[dev] = true;
  }
  p.pack = heads_in_tile(p.g);
  p.tile_tokens = f8::BM / p.pack;
  p.inv_pack = 65536 / p.pack + 1;  // exact for rows of a tile
  CUtensorMap mq, mk, mv;
  if (!make_tmap_3d(&mq, p.q, D, p.hq, total_q, D, p.q_stride, p.tile_tokens, p.pack)) return NVLLM_E_CUDA;
  const uint64_t slots = static_cast<uint64_t>(p.num_blocks) * kBlockSize;
  if (!make_tmap_codes(&mk, k_cache, D, p.hkv, slots, f8::BN) || !make_tmap_codes(&mv, v_cache, D, p.hkv, slots, f8::BN)) return NVLLM_E_CUDA;
  const int64_t items = prefill_fp8_items(p.hq, p.g, max_seqlen_q, p.batch);
  p.parts = workspace ? prefill_fp8_parts(items, max_seqlen_q, max_seqlen_k, prefill_fp8_blocks()) : 1;
  if (p.parts == 1) {
    const int grid = static_cast<int>(std::min<int64_t>(prefill_fp8_blocks(), items));
    return launch_kernel("prefill_fp8", prefill_fp8_kernel<D, false>, dim3(grid), dim3(f8::NTHREADS), G::SMEM, stream, p, mq, mk, mv);
  }
  const int grid = static_cast<int>(items) * p.parts;
  p.items = static_cast<int>(items);
  p.ws_items = reinterpret_cast<int4*>(static_cast<unsigned char*>(workspace) + kFp8CounterArea);
  p.ws_ml = reinterpret_cast<float2*>(p.ws_items + items);
  p.ws_o = reinterpret_cast<float4*>(p.ws_ml + static_cast<int64_t>(grid) * f8::BM);
  const int rc = launch_kernel("prefill_fp8", prefill_fp8_kernel<D, true>, dim3(grid), dim3(f8::NTHREADS), G::SMEM, stream, p, mq, mk, mv);
  if (rc) return rc;
  int log_rows = 0;  // of a tile, as far as they are there
  while ((1 << log_rows) < std::min(p.tile_tokens, max_seqlen_q) * p.pack) ++log_rows;
  const int64_t threads = (items * (D / 4)) << log_rows;
  return launch_kernel("prefill_fp8_join", prefill_fp8_join_kernel<D>, dim3(static_cast<unsigned>((threads + 255) / 256)), dim3(256), 0, stream,
                       p, log_rows);
}

}  // namespace nvllm

extern "C" int64_t nvllm_prefill_fp8_workspace_bytes(int32_t batch, int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_q_heads,
                                                     int32_t num_kv_heads, int32_t head_dim) {
  using namespace nvllm;
  if (batch < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads ||
      num_q_heads > 65535 || (head_dim != 64 && head_dim != 128))
    return fail(NVLLM_E_GEOMETRY, "prefill_fp8_workspace_bytes: batch=%d max_seqlen=%d / %d Hq=%d Hkv=%d head_dim=%d invalid", batch,
                max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads, head_dim);
  if (batch == 0 || max_seqlen_q == 0) return 0;
  const int64_t items = prefill_fp8_items(num_q_heads, num_q_heads / num_kv_heads, max_seqlen_q, batch);
  const int parts = prefill_fp8_parts(items, max_seqlen_q, max_seqlen_k, prefill_fp8_blocks());
  return parts == 1 ? 0 : kFp8CounterArea + items * 16 + items * parts * f8::BM * (head_dim + 2) * 4;
}

extern "C" int nvllm_prefill_varlen_fp8(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                                        const float* k_scale, const float* v_scale, const int32_t* block_tables,
                                        int64_t bt_row_stride, int32_t max_blocks, void* out, int64_t out_row_stride,
                                        const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int64_t total_q, int32_t batch,
                                        int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_q_heads, int32_t num_kv_heads,
                                        int32_t head_dim, float scale, int64_t num_blocks, void* workspace, int64_t workspace_bytes,
                                        void* stream) {
  using namespace nvllm;
  const char* who = "prefill_varlen_fp8";
  if (batch < 0 || max_seqlen_q < 0 || max_seqlen_k < 0 || total_q < 0)
    return fail(NVLLM_E_GEOMETRY, "%s: negative batch, max_seqlen or total_q", who);
  if (batch > f8::MAX_BATCH) return fail(NVLLM_E_GEOMETRY, "%s: batch=%d exceeds the %d sequences of one launch", who, batch, f8::MAX_BATCH);
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || num_q_heads > 65535)
    return fail(NVLLM_E_GEOMETRY, "%s: Hq=%d must be a positive multiple of Hkv=%d, at most 65535", who, num_q_heads, num_kv_heads);
  if (!(scale >= 0.f && scale < INFINITY)) return fail(NVLLM_E_GEOMETRY, "%s: scale must be finite and not negative", who);
  if (batch == 0 || max_seqlen_q == 0 || total_q == 0) return NVLLM_OK;
  const int rc = check_fp8_planes(who, k_cache, v_cache, k_scale, v_scale, num_kv_heads, head_dim, num_blocks);
  if (rc) return rc;
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || !block_tables) return fail(NVLLM_E_NULL, "%s: NULL pointer argument", who);
  const int64_t qrow = static_cast<int64_t>(num_q_heads) * head_dim;
  if (q_row_stride < qrow || out_row_stride < qrow || max_blocks <= 0 || bt_row_stride < max_blocks)
    return fail(NVLLM_E_GEOMETRY, "%s: a row stride is smaller than its row", who);
  if (static_cast<int64_t>(max_blocks) * kBlockSize > 0x7fffffffLL)
    return fail(NVLLM_E_GEOMETRY, "%s: max_blocks=%d too large", who, max_blocks);
  if (q_row_stride % 8 || out_row_stride % 8 || !aligned16(q) || !aligned16(out))
    return fail(NVLLM_E_ALIGN, "%s: q/out pointers and row strides must be 16-byte aligned", who);
  if (workspace) {
    const int64_t need = nvllm_prefill_fp8_workspace_bytes(batch, max_seqlen_q, max_seqlen_k, num_q_heads, num_kv_heads, head_dim);
    if (workspace_bytes < need)
      return fail(NVLLM_E_WORKSPACE, "%s: workspace of %lld bytes needed, %lld given", who, (long long)need, (long long)workspace_bytes);
    if (!aligned16(workspace)) return fail(NVLLM_E_ALIGN, "%s: workspace must be 16-byte aligned", who);
  }
  PrefillFp8Params p{};
  p.status = status_word();
  if (!p.status) return fail(NVLLM_E_NO_DEVICE, "%s: no CUDA device is usable", who);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_row_stride;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.bt_stride = bt_row_stride;
  p.max_blocks = max_blocks;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.out_stride = out_row_stride;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.batch = batch;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.g = num_q_heads / num_kv_heads;
  p.scale_log2e = scale * 1.4426950408889634f;
  p.num_blocks = num_blocks;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128) return launch_prefill_fp8<128>(p, k_cache, v_cache, total_q, max_seqlen_q, max_seqlen_k, workspace, st);
  return launch_prefill_fp8<64>(p, k_cache, v_cache, total_q, max_seqlen_q, max_seqlen_k, workspace, st);
}
