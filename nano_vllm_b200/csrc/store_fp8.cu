// store_kvcache_fp8: the new tokens' K/V rows to the 8-bit cache.
//
// For every group of 16 slots and KV head that rows go to, with f the lowest offset written and a the largest finite
// magnitude of the written rows of that head:
//   need = the smallest power of two with a <= 448 need;   scale = f == 0 ? need : max(need, scale)
//   written rows: code = e4m3(x / scale);  rows below f, where the scale has grown: code = e4m3(code * old / scale)
// f == 0 starts a group afresh (whatever an earlier owner of the block left in it counts for nothing); rows above f that are
// not written stay as they are, they belong to nobody yet.
//
// A warp owns a group and head of K or of V: it reads the group's rows once into registers (eight values a lane: 16 rows of 128
// take 32 registers, so that 24 warps of an SM have 100 KB on the way), takes the maximum by shuffles, and writes codes and
// scale, so no group is touched by two warps and nothing depends on their order.  The rows of a group stand next to each other
// in slot_mapping (rows that are skipped may lie between); the warp that the first of them falls to takes them all.
//
// 16384 rows of 8 heads of 128 (100 MB read and written) take 19 us; bytes alone are 15.6.  What binds is the integer unit (320 of
// a warp's 680 instructions, each two cycles of it): four values a lane and codes by way of fp32 were 22 us.  A resident block
// that goes on to the next rows instead of ending, with their slots loaded ahead, was 26: the chain from slots to rows to codes
// is hidden better by more blocks.
#include <algorithm>

#include "fp8.cuh"

namespace nvllm {

struct StoreFp8Params {
  const __nv_bfloat16* rows[2];  // K, V
  int64_t stride[2];
  unsigned char* cache[2];
  float* scale[2];
  const int32_t* slots;
  int64_t n;
  int64_t num_slots;
  int hkv;
  int near_rows;  // steps from row to row fit 32 bits
  int* status;
};

constexpr int kStoreFp8Threads = 256;
__device__ __forceinline__ int group_of(int slot) { return slot >> 4; }  // -1: none
static_assert(kScaleGroup == 16 && kGroups == 16);

// ALONE: one row to a block, for a step's rows, that are one to a group as a rule; otherwise 16.
template <int D, bool ALONE>
__global__ void __launch_bounds__(kStoreFp8Threads, ALONE ? 4 : 3) store_fp8_kernel(const StoreFp8Params p) {
  constexpr int LANES = D / 8;       // lanes that hold a row, eight values each
  constexpr int ROWS = 32 / LANES;   // rows that a warp takes at a time
  constexpr int ROWS_HERE = ALONE ? 1 : kScaleGroup;  // of a block
  constexpr int HELD = kScaleGroup / ROWS;
  constexpr unsigned ALL = 0xffffffffu;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int sub = lane / LANES, col = lane % LANES * 8;
  const bool is_v = blockIdx.y;
  const __nv_bfloat16* rows = (is_v ? p.rows[1] : p.rows[0]) + col;
  const int64_t stride = is_v ? p.stride[1] : p.stride[0];
  auto load = [&](int64_t r, int head) { return __ldg(reinterpret_cast<const uint4*>(rows + r * stride + head * D)); };

  pdl_wait();
  pdl_trigger();
  // The slots of this block's rows and of those behind them, a row to a lane, and of the 32 before; where a block has one row
  // its values come in the same trip.
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * ROWS_HERE, n_here = p.n - r0;
  const int raw = lane < n_here ? p.slots[r0 + lane] : -1, raw_before = r0 + lane >= 32 ? p.slots[r0 + lane - 32] : -1;
  uint4 early = make_uint4(0, 0, 0, 0);
  if (ALONE && sub == 0 && warp < p.hkv) early = load(r0, warp);
  if constexpr (!ALONE) {  // the block's rows to L2 while it finds out which of them go together
    constexpr int LINES = D / 64;  // of a row: 16 rows are 16 or 32 lines
    const int r = lane / LINES;
    if (r < kScaleGroup && r < n_here)
      for (int head = warp; head < p.hkv; head += warps)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(rows - col + (r0 + r) * stride + head * D + lane % LINES * 64));
  }
  auto stored = [&](int s) { return s < p.num_slots ? max(s, -1) : -1; };  // -1: nothing is stored
  const int slot = stored(raw);
  const bool own = lane < ROWS_HERE;
  if (warp == 0 && !is_v && own && raw >= p.num_slots) atomicOr(p.status, NVLLM_STATUS_BAD_SLOT);
  const unsigned live = __ballot_sync(ALL, slot >= 0);
  if (!__ballot_sync(ALL, own && slot >= 0)) return;
  // the group of the last stored row before this block's
  auto slot_at = [&](int64_t r) { return r >= 0 && r < p.n ? stored(p.slots[r]) : -1; };
  int before = -1, seen = stored(raw_before);
#pragma unroll 1
  for (int64_t r = r0 - 32; r > -32; r -= 32) {
    const unsigned m = __ballot_sync(ALL, seen >= 0);
    if (m) {
      before = group_of(__shfl_sync(ALL, seen, 31 - __clz(m)));
      break;
    }
    seen = slot_at(r - 32 + lane);
  }
  const int group = group_of(slot);
  const unsigned below = live & ((1u << lane) - 1);
  const int previous = __shfl_sync(ALL, group, below ? 31 - __clz(below) : lane);
  const unsigned leaders = __ballot_sync(ALL, own && slot >= 0 && group != (below ? previous : before));

#pragma unroll 1
  for (unsigned left = leaders; left; left &= left - 1) {
    const int at = __ffs(left) - 1;
    const int g = __shfl_sync(ALL, group, at);
    const int64_t i = r0 + at;
#pragma unroll 1
    for (int head = warp; head < p.hkv; head += warps) {
      // This lane's row of the next ROWS set bits of m, -1 if there is none.
      auto next_rows = [&](unsigned& m) {
        int b = -1;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
          const int bit = m ? __ffs(m) - 1 : -1;
          m &= m - 1;
          if (sub == k) b = bit;
        }
        return b;
      };
      // Where row b of the slots `sl` goes: rows in order, so that of several with the same slot the last one stays; of those at a
      // time none but it.
      auto destination = [&](int sl, int b) {
        const int to = __shfl_sync(ALL, sl, max(b, 0)), mine = b >= 0 ? to : -1;
        int last = mine;
#pragma unroll
        for (int k = 1; k < ROWS; ++k) {
          const int later = __shfl_down_sync(ALL, mine, k * LANES);
          if (sub + k < ROWS && later == mine) last = -1;
        }
        return last;
      };
      float* scale_at = (is_v ? p.scale[1] : p.scale[0]) + (static_cast<int64_t>(g >> 4) * p.hkv + head) * kGroups + (g & kGroups - 1);
      unsigned char* cache = (is_v ? p.cache[1] : p.cache[0]) + head * D + col;
      const int64_t row_bytes = static_cast<int64_t>(p.hkv) * D;
      auto code_at = [&](int to) { return reinterpret_cast<uint2*>(cache + to * row_bytes); };
      // The group's scale from the largest magnitude written (over the warp) and the scale so far, and the rows below `first` if it
      // has grown.  Returns its exponent.
      auto settle = [&](uint32_t most, int first, float old) {
        most = max(most & 0xffffu, most >> 16);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(ALL, most, d));
        const int e = first > 0 ? max(exponent_for(most), exponent_of(old)) : exponent_for(most);
        const float now = power_of_two(e);
        if (first > 0 && now != old) {
          const float ratio = old * power_of_two(-e);
#pragma unroll 1
          for (int r0 = sub; r0 < first; r0 += 4 * ROWS) {
            uint2 c[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (r0 + k * ROWS < first) c[k] = *code_at(g * kScaleGroup + r0 + k * ROWS);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (r0 + k * ROWS < first)
                *code_at(g * kScaleGroup + r0 + k * ROWS) = make_uint2(recode4(c[k].x, ratio), recode4(c[k].y, ratio));
          }
        }
        if (lane == 0) *scale_at = now;
        return e;
      };

      // Rows at + b of this group: bits b.
      const int behind = __shfl_sync(ALL, slot, (at + lane) & 31), sl = at + lane < 32 ? behind : -1;
      const unsigned same = __ballot_sync(ALL, sl >= 0 && group_of(sl) == g);
      const unsigned other = __ballot_sync(ALL, sl >= 0 && group_of(sl) != g);
      const unsigned run = other ? same & ((other & -other) - 1) : same;
      const bool ended = other != 0 || r0 + 32 >= p.n;  // a row of another group follows, or none
      const int first = __reduce_min_sync(ALL, run >> lane & 1u ? (sl & kScaleGroup - 1) : kScaleGroup);
      // Rows one after the other to slots one after the other, as sequences have them: all of them in registers.
      const int count = __popc(run), slot0 = __shfl_sync(ALL, slot, at);
      if (ended && p.near_rows && run == (2u << (count - 1)) - 1 && !__any_sync(ALL, lane < count && sl != slot0 + lane)) {
        float old = 0.f;
        if (first > 0) old = *scale_at;
        uint4 x[HELD];
        const uint4 none = make_uint4(0, 0, 0, 0);
        const unsigned char* from = reinterpret_cast<const unsigned char*>(rows + (i + sub) * stride + head * D);
        const uint32_t row_step = static_cast<uint32_t>(stride) * (2 * ROWS), code_step = static_cast<uint32_t>(row_bytes) * ROWS;
        auto row = [&](uint32_t j) { return __ldg(reinterpret_cast<const uint4*>(from + static_cast<uint64_t>(row_step) * j)); };
        const bool full = count == kScaleGroup;
        if (full) {
#pragma unroll
          for (int j = 0; j < HELD; ++j) x[j] = row(j);
        } else {
          const bool have = ALONE && head == warp;
          x[0] = have ? early : none;
          if (sub < count && !(have && sub == 0)) x[0] = row(0);
          if (count > ROWS) {
#pragma unroll
            for (int j = 1; j < HELD; ++j) x[j] = j * ROWS + sub < count ? row(j) : none;
          }
        }
        // two columns at a time; infinities and NaN stay what they are
        uint32_t most = max_magnitude(max_magnitude(x[0].x, x[0].y), max_magnitude(x[0].z, x[0].w));
        if (count > ROWS) {
#pragma unroll
          for (int j = 1; j < HELD; ++j)
            most = max_magnitude(max_magnitude(x[j].x, x[j].y), max_magnitude(max_magnitude(x[j].z, x[j].w), most));
        }
        most &= 0x7fff7fffu;
        if (!__any_sync(ALL, max(most & 0xffffu, most >> 16) >= 0x7f80u)) {
          const uint32_t inv = static_cast<uint32_t>(127 - settle(most, first, old)) * 0x00800080u;  // 2^-e as bf16, twice: exact
          unsigned char* to = cache + static_cast<int64_t>(slot0 + sub) * row_bytes;
          auto code = [&](uint32_t j) {
            *reinterpret_cast<uint2*>(to + static_cast<uint64_t>(code_step) * j) =
                make_uint2(encode4_finite(make_uint2(x[j].x, x[j].y), inv), encode4_finite(make_uint2(x[j].z, x[j].w), inv));
          };
          if (full) {
#pragma unroll
            for (int j = 0; j < HELD; ++j) code(j);
          } else {
            if (sub < count) code(0);
            if (count > ROWS) {
#pragma unroll
              for (int j = 1; j < HELD; ++j)
                if (j * ROWS + sub < count) code(j);
            }
          }
          continue;
        }
      }
      // Gaps, the same slots over and over, or something that is not finite: row by row, 32 slots at a time, as often as it takes.
      auto windows = [&](auto each) {
        int64_t from = i;
#pragma unroll 1
        while (true) {
          const int w = slot_at(from + lane);
          const unsigned in = __ballot_sync(ALL, w >= 0 && group_of(w) == g), out = __ballot_sync(ALL, w >= 0 && group_of(w) != g);
          unsigned m = out ? in & ((out & -out) - 1) : in;
          each(from, w, m);
          if (out != 0 || from + 32 >= p.n) break;
          from += 32;
        }
      };
      uint32_t most = 0;
      int lowest = kScaleGroup;
      windows([&](int64_t from, int w, unsigned m) {
        lowest = min(lowest, __reduce_min_sync(ALL, m >> lane & 1u ? (w & kScaleGroup - 1) : kScaleGroup));
#pragma unroll 1
        while (m) {
          const int b = next_rows(m);
          const uint4 v = b >= 0 ? load(from + b, head) : make_uint4(0, 0, 0, 0);
          most = max_finite2(max_finite2(max_finite2(max_finite2(most, v.x), v.y), v.z), v.w);
        }
      });
      const float inv = power_of_two(-settle(most, lowest, lowest > 0 ? *scale_at : 0.f));
      windows([&](int64_t from, int w, unsigned m) {
#pragma unroll 1
        while (m) {
          const int b = next_rows(m), to = destination(w, b);
          if (to >= 0) {
            const uint4 v = load(from + b, head);
            *code_at(to) = make_uint2(encode4(make_uint2(v.x, v.y), inv), encode4(make_uint2(v.z, v.w), inv));
          }
          __syncwarp();
        }
      });
    }
  }
}

}  // namespace nvllm

extern "C" int nvllm_store_kvcache_fp8(const void* key, int64_t key_row_stride, const void* value, int64_t value_row_stride,
                                       void* k_cache, void* v_cache, float* k_scale, float* v_scale,
                                       const int32_t* slot_mapping, int64_t n_tokens, int32_t num_kv_heads, int32_t head_dim,
                                       int64_t num_blocks, void* stream) {
  using namespace nvllm;
  if (n_tokens < 0) return fail(NVLLM_E_GEOMETRY, "store_kvcache_fp8: n_tokens=%lld < 0", (long long)n_tokens);
  if (n_tokens == 0) return NVLLM_OK;
  const int rc = check_fp8_planes("store_kvcache_fp8", k_cache, v_cache, k_scale, v_scale, num_kv_heads, head_dim, num_blocks);
  if (rc) return rc;
  if (!key || !value || !slot_mapping) return fail(NVLLM_E_NULL, "store_kvcache_fp8: NULL pointer argument");
  const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim;
  if (key_row_stride < row || value_row_stride < row)
    return fail(NVLLM_E_GEOMETRY, "store_kvcache_fp8: row strides (%lld, %lld) smaller than Hkv*D", (long long)key_row_stride,
                (long long)value_row_stride);
  if (key_row_stride % 8 || value_row_stride % 8 || !aligned16(key) || !aligned16(value))
    return fail(NVLLM_E_ALIGN, "store_kvcache_fp8: key/value pointers and row strides must be 16-byte aligned");
  StoreFp8Params p;
  p.status = status_word();
  if (!p.status) return fail(NVLLM_E_NO_DEVICE, "store_kvcache_fp8: no CUDA device is usable");
  p.rows[0] = static_cast<const __nv_bfloat16*>(key);
  p.rows[1] = static_cast<const __nv_bfloat16*>(value);
  p.stride[0] = key_row_stride;
  p.stride[1] = value_row_stride;
  p.cache[0] = static_cast<unsigned char*>(k_cache);
  p.cache[1] = static_cast<unsigned char*>(v_cache);
  p.scale[0] = k_scale;
  p.scale[1] = v_scale;
  p.slots = slot_mapping;
  p.n = n_tokens;
  p.num_slots = num_blocks * kBlockSize;
  p.hkv = num_kv_heads;
  p.near_rows = std::max({key_row_stride, value_row_stride, row}) < (int64_t{1} << 28);
  // Rows one to a group, as decode steps have them, want a row to a block (8 heads of 128, in a chain of launches: 250 rows 3.4 us,
  // 1000 rows 8.9), not a block that has up to 16 groups to do in turn (16.4, 16.5); rows of prompts want 16 to a block, which
  // finds a group's rows once (1000 rows 2.8, 2000 rows 3.9 us, 16000 rows 19; a row to a block: 6.1, 9.1, 72).  The slots are
  // on the device, so the number of rows decides: a step has no more than 1024 sequences as a rule.
  const bool alone = n_tokens <= 1024;
  const int64_t blocks = alone ? n_tokens : (n_tokens + kScaleGroup - 1) / kScaleGroup;
  if (blocks > 0x7fffffffLL) return fail(NVLLM_E_GEOMETRY, "store_kvcache_fp8: too many tokens for one launch");
  const int warps = std::min(num_kv_heads, kStoreFp8Threads / 32);
  const auto kernel = head_dim == 128 ? (alone ? store_fp8_kernel<128, true> : store_fp8_kernel<128, false>)
                                      : (alone ? store_fp8_kernel<64, true> : store_fp8_kernel<64, false>);
  return launch_kernel("store_kvcache_fp8", kernel, dim3(static_cast<unsigned>(blocks), 2), dim3(32 * warps), 0,
                       static_cast<cudaStream_t>(stream), p);
}
