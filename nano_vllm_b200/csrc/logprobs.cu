// Log probabilities of given tokens, entropy and top alternatives from rows of logits, in one pass.
//
// For a row of V logits x, temperature T (one that is not above 0 counts as 1), m = max x:
//   Z = sum exp((x_i - m) / T)            logprob of token k = (x_k - m) / T - ln Z
//   entropy = ln Z - sum exp((x_i - m) / T) (x_i - m) / T / Z
//   top alternatives: the `top` largest logits, ties to the lowest index, with their log probabilities
// The pass carries the running maximum and both sums, rescaled when the maximum grows.  A row with a NaN, with +infinity or
// with nothing but -infinity has no distribution: all its results are NaN (its alternatives go by the logits, NaN like -infinity).
//
// Alternatives without a second pass: a thread keeps the largest of its 16-byte pieces' maxima and the first piece that has it.
// Of 32 to 128 groups of threads the top-th largest (maximum, piece) is a bound that `top` elements reach, so every alternative lies
// in a thread whose own (maximum, piece) reaches it: about `top` threads, whose pieces are read again and compared with the bound
// (from L2 where the rows in flight fit in it; rows of 300 KB on every place of the device do not, and half of every sector of 32
// bytes that comes again from memory is for nothing).  Where those pieces are many, a thread keeps its largest for each segment of
// them.  Pieces break ties of values, and where many threads tie (a mask that leaves fewer than `top`) a block finds a closer bound
// among its own threads, counting the ties within their pieces.  Where more elements reach the bound than the list holds (largest
// ones that stand close together), each block keeps its own top ones.
//
// A row is read by a cluster of 1 to 8 blocks, four to a multiprocessor.
//
// What bounds it: 8 cycles of the unit for exponentials and about 7 issue slots an element and scheduler, beside 11 cycles of
// memory: of 4096 rows of 151936 bf16 the loads alone take 181 us, the pass 205-225, with one alternative 218 (5.7 TB/s; called one by
// one 254).  250 rows: 15.1, 20.8, with five 24.4 (500 blocks on 592 places).  One row with 20 alternatives: 7.4, of which the end 3:
// bound 0.4, listed threads' pieces 1.7, ranks and results 0.9, each a chain of short steps.  Rows of which a mask leaves 4 tokens,
// 20 alternatives: one 10.3, 64 23 (13 without a mask), 250 28 (27.5); 64 alternatives: 2000 rows of 1000 26 (24).
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "logprobs.cuh"

namespace nvllm {

constexpr int kLpThreads = 256;
template <bool TOP>
constexpr int kLpStep = TOP ? 3 : 4;  // pieces that a thread takes at a time
constexpr int kLpMaxCluster = 8;
constexpr int kLpMaxTop = NVLLM_LOGPROBS_MAX_TOP;
constexpr int kLpGroups = 128;   // of threads, whose maxima give the bound
constexpr int kLpTied = 8;       // threads at the bound's value that make a block look for a closer one (4 and 16 measured the same)
constexpr int kLpSegments = 8;   // of a thread's pieces, at most
constexpr int kLpCands = 1024;   // elements that reach the bound, as many as the list holds

struct LogprobParams {
  const void* logits;
  int64_t row_stride;
  const int64_t* tokens;
  const float* temperatures;  // nullable
  int vocab, top;
  int groups;  // of the threads that read a row, whose maxima give the bound: 32 to 128
  int log_csize, log_all, log_size;  // blocks of a row, its threads, threads of a group: powers of two, divided by with shifts
  int log_seg;  // steps of a segment (PARTED)
  float* logprobs;
  float* entropy;
  int64_t* top_tokens;
  float* top_logprobs;
  int* status;
};

// Float as an unsigned number of the same order; NaN like -infinity, one zero, subnormal numbers (to which comparisons are
// blind, as this is compiled) like it.
__device__ __forceinline__ uint32_t lp_order(float x) {
  uint32_t u = __float_as_uint(x);
  if ((u & 0x7fffffffu) > 0x7f800000u) u = 0xff800000u;
  if (!(u & 0x7f800000u)) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
// Orders by value, then lower place first.  Never 0.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t place) { return (static_cast<uint64_t>(lp_order(x)) << 32) | (0xffffffffu - place); }

// 16 bytes of a row.
template <typename T>
struct LpPiece;
template <>
struct LpPiece<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[N]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float max(const uint4& w) {  // NaN ignored
    auto h = [](uint32_t u) { return *reinterpret_cast<__nv_bfloat162*>(&u); };
    const __nv_bfloat162 m = __hmax2(__hmax2(h(w.x), h(w.y)), __hmax2(h(w.z), h(w.w)));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    auto f = [](uint32_t u, uint32_t v) {
      const __nv_bfloat162 m = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&u), *reinterpret_cast<__nv_bfloat162*>(&v));
      return *reinterpret_cast<const uint32_t*>(&m);
    };
    return make_uint4(f(a.x, b.x), f(a.y, b.y), f(a.z, b.z), f(a.w, b.w));
  }
  static __device__ __forceinline__ float max_or_nan(const uint4& w) {
    auto f = [](uint32_t u, uint32_t v) {
      uint32_t r;
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(v));
      return r;
    };
    const uint32_t m = f(f(w.x, w.y), f(w.z, w.w));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  // -infinity becomes the lowest finite number, NaN stays
  static __device__ __forceinline__ uint4 lift(const uint4& w) {
    auto f = [](uint32_t u) {
      uint32_t r;
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(u), "r"(0xff7fff7fu));
      return r;
    };
    return make_uint4(f(w.x), f(w.y), f(w.z), f(w.w));
  }
  // -infinity in the places below lo and from hi on
  static __device__ __forceinline__ uint4 cut(uint4 w, int lo, int hi) {
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < lo || k >= hi) u[k / 2] = k % 2 ? (u[k / 2] & 0xffffu) | 0xff800000u : (u[k / 2] & 0xffff0000u) | 0xff80u;
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <>
struct LpPiece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& w, float (&x)[N]) {
    x[0] = __uint_as_float(w.x);
    x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z);
    x[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ float max(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ float max_or_nan(const uint4& w) {
    return max_nan(max_nan(__uint_as_float(w.x), __uint_as_float(w.y)), max_nan(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ uint4 lift(const uint4& w) {
    auto f = [](uint32_t u) { return __float_as_uint(max_nan(__uint_as_float(u), -FLT_MAX)); };
    return make_uint4(f(w.x), f(w.y), f(w.z), f(w.w));
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    auto f = [](uint32_t u, uint32_t v) { return __float_as_uint(fmaxf(__uint_as_float(u), __uint_as_float(v))); };
    return make_uint4(f(a.x, b.x), f(a.y, b.y), f(a.z, b.z), f(a.w, b.w));
  }
  static __device__ __forceinline__ uint4 cut(uint4 w, int lo, int hi) {
    uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k < lo || k >= hi) u[k] = 0xff800000u;
    return make_uint4(u[0], u[1], u[2], u[3]);
  }
};

extern __shared__ uint64_t s_seg[];  // [kLpSegments][threads]: the largest (maximum, piece) of a segment

// From the threads' statistics to the row's results.
template <typename T, bool TOP, bool PARTED>
__device__ __noinline__ void lp_finish(const float sum_m, const float sum_s, const float sum_t, const uint64_t mine, const uint4* const base,
                                       const int shift, const int pieces, const int head, const int tail, const float inv_t, const float given,
                                       const int64_t token, const int vocab, const int top, const int groups, const int log_csize, const int log_all,
                                       const int log_size, const int log_seg, float* const logprobs, float* const entropy, int64_t* const top_tokens,
                                       float* const top_logprobs, int* const status) {
  using P = LpPiece<T>;
  constexpr int N = P::N, C = kLpStep<TOP>;
  namespace cg = cooperative_groups;
  __shared__ __align__(16) uint64_t s_bounds[kLpGroups];
  __shared__ uint64_t s_cand[kLpCands];  // of the first block
  __shared__ float s_sums[kLpMaxCluster][3];
  __shared__ float s_warp[kLpThreads / 32][3];
  __shared__ uint16_t s_slot[kLpThreads], s_part[PARTED ? 2 * kLpMaxTop * kLpSegments : 1];
  __shared__ __align__(16) uint64_t s_key[kLpThreads];
  __shared__ uint64_t s_tau;
  __shared__ float s_m, s_log_z;
  __shared__ int s_slots, s_parts, s_cands, s_reach[2][kLpThreads / 32];
  const cg::cluster_group cluster = cg::this_cluster();
  const int csize = 1 << log_csize, crank = blockIdx.x & (csize - 1), row = blockIdx.x >> log_csize;
  const bool several = csize > 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = 1 << (log_all - log_csize), all = 1 << log_all, me = crank * threads + tid;
  const int whole = pieces - head - tail;
  const float c = inv_t * 1.4426950408889634f;
  LpSums sum{sum_m, sum_s, sum_t};
  if (tid == 0) {
    s_tau = 0;
    s_slots = s_parts = s_cands = 0;
  }
  // ---- sums of the block, and the largest (maximum, piece) of every group of threads
  auto join_warp = [&](LpSums& v) {  // over the lanes
    float m = v.m;
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, sh));
    v.rescale(m, c);
#pragma unroll
    for (int sh = 16; sh > 0; sh >>= 1) {
      v.s += __shfl_xor_sync(0xffffffffu, v.s, sh);
      v.t += __shfl_xor_sync(0xffffffffu, v.t, sh);
    }
  };
  join_warp(sum);
  if (lane == 0) {
    s_warp[warp][0] = sum.m;
    s_warp[warp][1] = sum.s;
    s_warp[warp][2] = sum.t;
  }
  auto sync = [&]() {
    if (several) cluster.sync();
    else __syncthreads();
  };
  if (several) cluster.barrier_wait();
  if constexpr (TOP) {
    const int size = 1 << log_size;  // threads of a group: 1 to 32
    uint64_t most = mine;
    for (int sh = 1; sh < size; sh <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, sh));
    // every block of the row gets all groups'
    for (int to = tid & (size - 1); to < csize; to += size) (several ? cluster.map_shared_rank(s_bounds, to) : s_bounds)[me >> log_size] = most;
  }
  __syncthreads();
  if (warp == 0) {
    const int w = min(lane, threads / 32 - 1);
    sum = {s_warp[w][0], lane == w ? s_warp[w][1] : 0.f, lane == w ? s_warp[w][2] : 0.f};
    join_warp(sum);
    if (lane == 0) {
      float* to = (several ? cluster.map_shared_rank(&s_sums[0][0], 0) : &s_sums[0][0]) + 3 * crank;
      to[0] = sum.m;
      to[1] = sum.s;
      to[2] = sum.t;
    }
  }
  pdl_trigger();
  sync();

  // ---- the bound that `top` elements of the row reach, and the elements that do: to the first block's list
  int* cands_at = several ? cluster.map_shared_rank(&s_cands, 0) : &s_cands;
  uint64_t* cand_at = several ? cluster.map_shared_rank(s_cand, 0) : s_cand;
  uint64_t tau = 0;
  float each_inv = 0.f;
  int each = 0, total = 0, looked = 0;
  // The keys of the elements that reach the bound in piece n of what is listed (a thread, or a segment of one), 0 in the place of the others.
  auto look = [&](int n, uint64_t (&keys)[N]) {
#pragma unroll
    for (int k = 0; k < N; ++k) keys[k] = 0;
    int g;
    uint4 w;
    if (n < total) {
      const int nth = static_cast<int>((static_cast<float>(n) + 0.5f) * each_inv);
      if constexpr (PARTED) g = head + crank * threads + s_part[nth] % kLpThreads + (s_part[nth] / kLpThreads * each + n - nth * each) * all;
      else g = head + crank * threads + s_slot[nth] + (n - nth * each) * all;
      if (g >= head + whole) return;
      w = __ldg(base + g);
    } else if (n < looked) {  // the cut pieces, whether they are in a listed thread or not
      g = n == total && head ? 0 : pieces - 1;
      const int last_hi = shift + vocab - (pieces - 1) * N;
      w = P::cut(__ldg(base + g), g == 0 ? shift : 0, g == pieces - 1 ? last_hi : N);
    } else {
      return;
    }
    float e[N];
    P::unpack(w, e);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int id = g * N + k - shift;
      if (id >= 0 && id < vocab && lp_key(e[k], static_cast<uint32_t>(g)) >= tau) keys[k] = lp_key(e[k], static_cast<uint32_t>(id));
    }
  };
  // Elements that reach the bound, and `least`, to the first block's list.
  auto collect = [&](uint64_t least) {
    for (int n = tid; n < looked; n += threads) {
      uint64_t keys[N];
      look(n, keys);
      int found = 0;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        if (keys[k] < least) keys[k] = 0;
        found += keys[k] != 0;
      }
      if (!found) continue;
      int place = atomicAdd(cands_at, found);  // one for a piece: 0.2 us each at another block
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (keys[k]) {
          if (place < kLpCands) cand_at[place] = keys[k];
          ++place;
        }
    }
  };
  if constexpr (TOP) {
    // how many groups are above one: two threads count
    const ulonglong2* bounds = reinterpret_cast<const ulonglong2*>(s_bounds);
    for (int n = tid / 2; n < groups; n += threads / 2) {
      const uint64_t it = s_bounds[n];
      int above = 0;
#pragma unroll 8
      for (int k = tid % 2; k < groups / 2; k += 2) {
        const ulonglong2 v = bounds[k];
        above += (v.x > it) + (v.y > it);
      }
      above += __shfl_xor_sync(0xffffffffu, above, 1);
      if (tid % 2 == 0 && above == top - 1 && it) s_tau = it;  // one group: keys differ
    }
    __syncthreads();
    tau = s_tau;
    auto list = [&]() {
      if (mine && mine >= tau) {
        const int k = atomicAdd(&s_slots, 1);
        s_slot[k] = static_cast<uint16_t>(tid);
        s_key[k] = mine;
      }
      return __syncthreads_count(mine && mine >= tau && mine >> 32 == tau >> 32);  // threads whose largest is the bound's value
    };
    const int tied = list();
    if (s_slots > 2 * top || tied > kLpTied) {
      // A closer bound among the block's own threads.  Of a thread with (value, piece), so many elements reach that: those of the value in
      // the piece, of a masked one all.  The bound is where these numbers, from the largest key on, come to `top`.  (Without the numbers, each
      // thread for one element: 250 rows of which 4 tokens are left, 20 alternatives, 53 us instead of 33; 64 of 64 alternatives 425 instead
      // of 34; with 5 alternatives 21.8 instead of 22.4.)  Places are below 2^23: they move up four bits to make room.
      const int n = s_slots;
      const uint64_t it = tid < n ? s_key[tid] : 0;
      uint64_t mark = 0;
      int ties = 1;
      if (it) {
        const int g = static_cast<int>(0xffffffffu - static_cast<uint32_t>(it));
        if (g >= head && g < head + whole) {
          float e[N];
          P::unpack(__ldg(base + g), e);
          ties = 0;
#pragma unroll
          for (int k = 0; k < N; ++k) ties += lp_order(e[k]) == static_cast<uint32_t>(it >> 32);
        }
        ties = max(ties, 1);
        mark = (it >> 32 << 32) | (static_cast<uint32_t>(it) << 4) | ties;
      }
      s_key[tid] = mark;
      __syncthreads();
      int above = 0;
      const ulonglong2* marks = reinterpret_cast<const ulonglong2*>(s_key);
      for (int k = 0; k < n; k += 8) {
        ulonglong2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = marks[k / 2 + i];
#pragma unroll
        for (int i = 0; i < 4; ++i) above += (v[i].x > mark ? static_cast<int>(v[i].x & 15) : 0) + (v[i].y > mark ? static_cast<int>(v[i].y & 15) : 0);
      }
      if (it && above < top && above + ties >= top) s_tau = it;
      if (tid == 0) s_slots = 0;
      __syncthreads();
      tau = s_tau;
      list();
    }
    int listed = s_slots;
    each = (whole + all - 1) >> log_all;  // pieces of a thread
    if constexpr (PARTED) {               // of the listed threads the segments that reach the bound
      each = C << log_seg;
      for (int n = tid; n < listed * kLpSegments; n += threads) {
        const int who = s_slot[n / kLpSegments], part = n % kLpSegments;
        if (s_seg[part * threads + who] >= tau) s_part[atomicAdd(&s_parts, 1)] = static_cast<uint16_t>(part * kLpThreads + who);
      }
      __syncthreads();
      listed = s_parts;
    }
    each_inv = __frcp_rn(static_cast<float>(each));
    total = listed * each;
    looked = total + (crank == 0 ? head + tail : 0);
    collect(0);
  }
  if (crank == 0 && warp == threads / 32 - 1) {  // the warp with least to look at
    const int b = min(lane, csize - 1);
    sum = {s_sums[b][0], lane == b ? s_sums[b][1] : 0.f, lane == b ? s_sums[b][2] : 0.f};
    join_warp(sum);
    if (lane == 0) {
      const float log_z = sum.log_z();
      s_log_z = log_z;
      s_m = sum.m;
      sum.results(row, token, given, inv_t, log_z, vocab, logprobs, entropy, status);
    }
  }
  if constexpr (!TOP) return;
  sync();
  int cands = *cands_at;
  if (cands > kLpCands) {
    // Of a block no more than `top` go on: those that reach the key that `top` of its keys reach, which is found bit by bit (places are
    // below 2^24, so eight bits are known).  151936 ascending logits, 64 alternatives: 34 us.
    uint64_t least = 0;
    for (int bit = 63; bit >= 0; --bit) {
      if (bit == 31) {
        least |= 0xff000000u;
        bit = 23;
      }
      const uint64_t to = least | 1ull << bit;
      int count = 0;
      for (int n = tid; n < looked; n += threads) {
        uint64_t keys[N];
        look(n, keys);
#pragma unroll
        for (int k = 0; k < N; ++k) count += keys[k] >= to;
      }
      count = __reduce_add_sync(0xffffffffu, count);
      if (lane == 0) s_reach[bit & 1][warp] = count;
      __syncthreads();
      count = 0;
      for (int w = 0; w < threads / 32; ++w) count += s_reach[bit & 1][w];
      if (count >= top) least = to;
      if (count == top) break;
    }
    sync();
    if (crank == 0 && tid == 0) s_cands = 0;
    sync();
    collect(least);
    sync();
    cands = *cands_at;
  }
  if (several) cluster.barrier_arrive();  // the first block's counter has been read
  if (crank == 0) {
    // ranks by counting, eight threads a candidate
    for (int n = tid / 8; n < ((cands + 3) & ~3); n += threads / 8) {
      const uint64_t key = n < cands ? s_cand[n] : 0;
      int rank = 0;
#pragma unroll 4
      for (int k = tid % 8; k < cands; k += 8) rank += s_cand[k] > key;
#pragma unroll
      for (int sh = 1; sh < 8; sh <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, sh);
      if (tid % 8 == 0 && n < cands && rank < top) {
        const int64_t to = static_cast<int64_t>(row) * top + rank;
        top_tokens[to] = 0xffffffffu - static_cast<uint32_t>(key);
        top_logprobs[to] = (lp_value(static_cast<uint32_t>(key >> 32)) - s_m) * inv_t - s_log_z;
      }
    }
  }
  if (several) cluster.barrier_wait();
}

template <typename T, bool TOP, bool PARTED>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(const __grid_constant__ LogprobParams p) {
  using P = LpPiece<T>;
  constexpr int N = P::N, C = kLpStep<TOP>;
  pdl_wait();
  const int csize = 1 << p.log_csize, crank = blockIdx.x & (csize - 1);
  const bool several = csize > 1;
  if (several) cooperative_groups::this_cluster().barrier_arrive();  // waited for before another block's shared memory is written
  const int row = blockIdx.x >> p.log_csize, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = 1 << (p.log_all - p.log_csize);
  const int me = crank * threads + tid, all = 1 << p.log_all;  // of the row's threads
  const T* x = static_cast<const T*>(p.logits) + static_cast<int64_t>(row) * p.row_stride;

  // Pieces start on 16-byte boundaries: what lies before and behind the row in the first and last one counts as -infinity.
  const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
  const uint4* base = reinterpret_cast<const uint4*>(x - shift);
  const int pieces = static_cast<int>((static_cast<int64_t>(shift) + p.vocab + N - 1) / N);
  const int last_hi = shift + p.vocab - (pieces - 1) * N;  // places of the last piece
  const int head = shift > 0 || pieces == 1 ? 1 : 0;       // piece 0 is cut: the row's first thread has it
  const int tail = pieces > 1 && last_hi < N ? 1 : 0;      // and the last one
  const int whole = pieces - head - tail;
  auto cut_piece = [&](int g) { return P::cut(__ldg(base + g), g == 0 ? shift : 0, g == pieces - 1 ? last_hi : N); };

  // A thread takes C pieces at a time; those of the next step are loaded before the current ones are looked at, into the other of
  // two sets of registers (one set, copied, took 0.5 instructions an element).  The last step, which not all pieces may have, comes
  // first, beside the first one.
  const uint4* from = base + head;
  const int step = C * all;
  const int steps = max(0, ((whole - (me - lane) - 32 + all) >> p.log_all) / C);  // that all lanes have whole
  const int rest = me + steps * step;                                                   // where the last one starts
  uint4 x0[C], x1[C];
  auto load = [&](uint4 (&to)[C], int j) {
#pragma unroll
    for (int k = 0; k < C; ++k) to[k] = __ldg(from + j + k * all);
  };
  if (steps > 0) load(x0, me);
  const uint4 nothing = P::cut(make_uint4(0, 0, 0, 0), 0, 0);
#pragma unroll
  for (int k = 0; k < C; ++k) x1[k] = rest + k * all < whole ? __ldg(from + rest + k * all) : nothing;
  const float inv_t = lp_inverse(p.temperatures, row);
  const float c = inv_t * 1.4426950408889634f;
  int64_t token = -1;
  float given = 0.f;
  if (crank == 0 && tid == threads - 32) {  // which writes the results
    token = p.tokens[row];
    if (token >= 0 && token < p.vocab) given = static_cast<float>(x[token]);
  }

  LpSums sum{-FLT_MAX, 0.f, 0.f};
  float best = -INFINITY;
  const bool any = me == 0 || me < whole;
  int at = 0;  // the first piece with the largest element so far
  const uint64_t c2 = pack2(c, c);
  // Sums over pieces.  A masked element's difference is -infinity, whose product with its weight of 0 is NaN.  A warp that comes upon
  // one lifts -infinity to the lowest finite number first, from then on: half an instruction an element, pieces of which nothing is
  // left are passed over, and the sums are right while the maximum is far above that number and differences do not overflow;
  // otherwise the pieces are read again and summed one by one, with the differences kept finite.
  bool masked = false;
  auto add = [&](const uint4& w, auto finite, uint64_t& s2, uint64_t& t2) {
    const uint64_t minus_m = pack2(-sum.m, -sum.m);
    float e[N];
    P::unpack(w, e);
#pragma unroll
    for (int k = 0; k < N; k += 2) {
      uint64_t y = add2(pack2(e[k], e[k + 1]), minus_m);
      float a, b;
      if constexpr (decltype(finite)::value) {
        unpack2(y, a, b);
        y = pack2(max_nan(a, -3e38f), max_nan(b, -3e38f));
      }
      unpack2(mul2(y, c2), a, b);
      const uint64_t w2 = pack2(fast_exp2(a), fast_exp2(b));
      s2 = add2(s2, w2);
      t2 = fma2(w2, y, t2);
    }
  };
  auto one = [&](const uint4& w) {
    uint64_t s2 = 0, t2 = 0;
    add(w, std::true_type{}, s2, t2);
    float a, b;
    unpack2(s2, a, b);
    sum.s += a + b;
    unpack2(t2, a, b);
    sum.t += a + b;
  };
  // The maximum in use is the warp's: that grows a few times a row, a lane's in nearly every step of some lane.
  auto grow = [&](float most) {
    if (__any_sync(0xffffffffu, most > sum.m)) {
      float m = fmaxf(most, sum.m);
#pragma unroll
      for (int sh = 16; sh > 0; sh >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, sh));
      sum.rescale(m, c);
    }
  };
  // Pieces i, i + all, ...; ragged: some of them may not be there.
  auto take = [&](uint4 (&raw)[C], int i, bool ragged) {
    if constexpr (TOP) {
      float largest = -INFINITY;
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const float most = P::max(raw[k]);
        if (most > best) {
          best = most;
          at = head + i + k * all;
        }
        largest = fmaxf(largest, most);
      }
      grow(largest);
    } else {
      uint4 m = raw[0];
#pragma unroll
      for (int k = 1; k < C; ++k) m = P::larger(m, raw[k]);
      grow(P::max(m));
    }
    bool lifted = masked || ragged;
    while (true) {
      if (lifted) {
        float most = P::max_or_nan(raw[0]);
#pragma unroll
        for (int k = 1; k < C; ++k) most = max_nan(most, P::max_or_nan(raw[k]));
        if (__all_sync(0xffffffffu, most == -INFINITY)) return;  // nothing left of them
#pragma unroll
        for (int k = 0; k < C; ++k) raw[k] = P::lift(raw[k]);
      }
      uint64_t s2 = 0, t2 = 0;
#pragma unroll
      for (int k = 0; k < C; ++k) add(raw[k], std::false_type{}, s2, t2);
      float a, b, u, v;
      unpack2(s2, a, b);
      unpack2(t2, u, v);
      u += v;
      if (!__any_sync(0xffffffffu, u != u || (lifted && sum.m < -3e38f))) {
        sum.s += a + b;
        sum.t += u;
        return;
      }
      if (lifted) break;
      lifted = masked = true;
    }
#pragma unroll 1
    for (int k = 0; k < C; ++k)
      if (i + k * all < whole) one(__ldg(from + i + k * all));
  };
  if (rest - lane < whole) {
    at = head + rest;
    take(x1, rest, true);
  }
  const float best_last = best;
  const int at_last = !PARTED || rest < whole ? at : -1;
  best = -INFINITY;
  at = head + me;
  if constexpr (PARTED)  // segments without a piece
    for (int k = steps >> p.log_seg; k < kLpSegments; ++k) s_seg[k * threads + tid] = 0;
  for (int n = 0, i = me; n < steps; n += 2) {
    if (n + 1 < steps) load(x1, i + step);
    take(x0, i, false);
    i += step;
    if (n + 1 >= steps) break;
    if (n + 2 < steps) load(x0, i + step);
    take(x1, i, false);
    i += step;
    if constexpr (PARTED) {
      if (((n + 2) >> p.log_seg) != (n >> p.log_seg)) {
        s_seg[(n >> p.log_seg) * threads + tid] = lp_key(best, static_cast<uint32_t>(at));
        best = -INFINITY;
        at = head + i;
      }
    }
  }
  bool open = steps > 0;  // the loop has left pieces that are in no segment yet
  if constexpr (PARTED) open = steps >> p.log_seg << p.log_seg != steps;
  if (best_last > best || !open) {
    best = best_last;
    at = at_last;
  }
  uint64_t others = 0;
  if constexpr (PARTED) {
    if (at >= 0) s_seg[(steps >> p.log_seg) * threads + tid] = lp_key(best, static_cast<uint32_t>(at));
    for (int k = 0; k < steps >> p.log_seg; ++k) others = max(others, s_seg[k * threads + tid]);
  }
  if (crank == 0 && warp == 0 && (head || tail)) {
    const uint4 w0 = head && lane == 0 ? cut_piece(0) : nothing, w1 = tail && lane == 0 ? cut_piece(pieces - 1) : nothing;
    const float first = P::max(w0), last = P::max(w1);
    if (head && lane == 0 && !(first < best)) {  // the lowest piece, whenever it is looked at
      best = fmaxf(first, -INFINITY);
      at = 0;
    }
    if (last > best) {
      best = last;
      at = pieces - 1;
    }
    grow(fmaxf(first, last));
    one(w0);
    one(w1);
  }

  // What the end of a row wants of registers would cost the stream a tenth if it were part of it.
  uint64_t mine = any ? lp_key(best, static_cast<uint32_t>(at)) : 0;
  if constexpr (PARTED) mine = at >= 0 ? max(others, mine) : others;
  lp_finish<T, TOP, PARTED>(sum.m, sum.s, sum.t, mine, base, shift, pieces, head, tail, inv_t, given, token, p.vocab, p.top,
                    p.groups, p.log_csize, p.log_all, p.log_size, p.log_seg, p.logprobs, p.entropy, p.top_tokens, p.top_logprobs, p.status);
}

}  // namespace nvllm

extern "C" int nvllm_token_logprobs(const void* logits, int32_t logits_are_fp32, int64_t row_stride, const int64_t* tokens,
                                    const float* temperatures, int32_t rows, int32_t vocab, int32_t top, float* logprobs,
                                    float* entropy, int64_t* top_tokens, float* top_logprobs, void* stream) {
  using namespace nvllm;
  // a listed piece's thread is found by a product in fp32, which is right for up to 2^22 pieces of a block's 2 top listed threads
  if (rows < 0 || vocab <= 0 || vocab > NVLLM_LOGPROBS_MAX_VOCAB)
    return fail(NVLLM_E_GEOMETRY, "token_logprobs: rows=%d vocab=%d (1 to %d) not supported", rows, vocab, NVLLM_LOGPROBS_MAX_VOCAB);
  if (top < 0 || top > kLpMaxTop || top > vocab)
    return fail(NVLLM_E_GEOMETRY, "token_logprobs: top=%d outside 0 to %d (vocab=%d)", top, kLpMaxTop, vocab);
  if (rows == 0) return NVLLM_OK;
  if (!logits || !tokens || !logprobs || !entropy || (top > 0 && (!top_tokens || !top_logprobs)))
    return fail(NVLLM_E_NULL, "token_logprobs: NULL pointer argument");
  if (row_stride < vocab) return fail(NVLLM_E_GEOMETRY, "token_logprobs: the row stride is smaller than vocab");
  auto off = [](const void* q, size_t n) { return reinterpret_cast<uintptr_t>(q) % n != 0; };
  if (off(logits, logits_are_fp32 ? 4 : 2) || off(tokens, 8) || off(temperatures, 4) || off(logprobs, 4) || off(entropy, 4) ||
      off(top_tokens, 8) || off(top_logprobs, 4))
    return fail(NVLLM_E_ALIGN, "token_logprobs: a pointer is not aligned to its element size");
  LogprobParams p;
  p.status = status_word();
  const int sms = num_sms();
  if (!p.status || sms <= 0) return fail(NVLLM_E_NO_DEVICE, "token_logprobs: no CUDA device is usable");
  p.logits = logits;
  p.row_stride = row_stride;
  p.tokens = tokens;
  p.temperatures = temperatures;
  p.vocab = vocab;
  p.top = top;
  p.logprobs = logprobs;
  p.entropy = entropy;
  p.top_tokens = top_tokens;
  p.top_logprobs = top_logprobs;
  const int64_t pieces = (static_cast<int64_t>(vocab) + (logits_are_fp32 ? 3 : 7)) / (logits_are_fp32 ? 4 : 8);
  // Blocks of a row: as many as the device holds at a time with four to a multiprocessor, each thread with two pieces or more (one row
  // in one block 20.7 us, two 13.8, four 9.6, eight 8.4; 250 rows in one 33, two 28, four 35).  Threads of a row of its own block: eight
  // pieces each (5000 rows of 100 in blocks of 64 threads 60 us, 256 79; 4096 of 32000 in 64 162, 256 110), but twice as many as there are
  // alternatives, as long as they have a piece: with fewer the bound is loose (64 alternatives, 2000 rows of 1000 in 64 threads 81 us, 128 24;
  // 4096 of 4000 161 and 60; with a mask that leaves 4 tokens 2000 of 1000 20.5 and 28).
  int csize = kLpMaxCluster, threads = kLpThreads;
  while (csize > 1 && (static_cast<int64_t>(rows) * csize > 4ll * sms || pieces < 2ll * csize * kLpThreads)) csize /= 2;
  while (csize == 1 && threads > 64 && pieces < 8ll * threads && std::min<int64_t>(2 * top, pieces) <= threads / 2) threads /= 2;
  const int all = csize * threads;
  // Groups: 2.5 for each alternative, so that the bound lies close to the last one; more take longer to be counted against one another.
  // In 32, 64 and 128 groups: 250 rows of 151643 with 5 alternatives 24.4, 24.6, 25.5 us, 12 25.8, 25.9, 26.8, 16 27.1, 26.7, 27.3, 24 30.9,
  // 28.5, 28.8, 40 -, 29.6, 29.3; 2000 of 32000 with 12 44.1, 43.3, 46.1, 24 55.3, 50.4, 51.8, 32 68, 56.2, 57.1, 40 -, 63.4, 60.1; a cluster's 64
  // and 128: 64 fp32 rows with 24 15.3, 15.4, 32 16.6, 15.9.  And as many pieces to a group as there are alternatives to be told apart.
  p.groups = std::max(32, all / 32);
  while (p.groups < std::min(kLpGroups, all) && (2 * p.groups < 5 * top || pieces * p.groups < static_cast<int64_t>(top) * all)) p.groups *= 2;
  auto log2_of = [](int n) {
    int l = 0;
    while (n >> (l + 1)) ++l;
    return l;
  };
  p.log_csize = log2_of(csize);
  p.log_all = log2_of(all);
  p.log_size = log2_of(all / p.groups);
  // Segments of a thread's pieces, so that some and not all pieces of a listed thread are read again: where those would be more than two for
  // each thread, of 32 or more (4096 rows of 151936 with 20 alternatives 320 us, in segments 272; with five 231 and 261; 300 rows with 64 76 and 47;
  // 1003 fp32 rows with 64 219 and 147).  The pass itself takes 218 us without and 250 with them.
  const int64_t each = (pieces + all) / all, steps = each / kLpStep<true> + 1;
  const bool parted = each >= 32 && top * each > 2 * all;
  p.log_seg = 1;
  while (steps >> p.log_seg >= kLpSegments) ++p.log_seg;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows * csize), 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = parted ? kLpSegments * threads * sizeof(uint64_t) : 0;
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = csize;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = csize > 1 ? 2 : 1;
  auto of = [&](auto type) {
    using T = decltype(type);
    return parted ? logprobs_kernel<T, true, true> : top > 0 ? logprobs_kernel<T, true, false> : logprobs_kernel<T, false, false>;
  };
  auto kernel = logits_are_fp32 ? of(0.f) : of(__nv_bfloat16());
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(NVLLM_E_CUDA, "token_logprobs launch: %s", cudaGetErrorString(e));
  }
  count_launch();
  return NVLLM_OK;
}
