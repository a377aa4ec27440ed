// store_kvcache_fp8: the new tokens' K/V rows to the 8-bit cache.
//
// For every group of 16 slots and KV head that rows go to, with f the lowest offset written and a the largest finite
// magnitude of the written rows of that head:
//   need = the smallest power of two with a <= 448 need;   scale = f == 0 ? need : max(need, scale)
//   written rows: code = e4m3(x / scale);  rows below f, where the scale has grown: code = e4m3(code * old / scale)
// f == 0 starts a group afresh (whatever an earlier owner of the block left in it counts for nothing); rows above f that are
// not written stay as they are, they belong to nobody yet.
//
// A warp owns a group and head: it reads the group's rows once into registers (16 rows of K by one half of the warp, of V by
// the other), takes the maximum by shuffles, and writes codes and scale, so no group is touched by two warps and nothing
// depends on their order.  The rows of a group stand next to each other in slot_mapping (rows that are skipped may lie between);
// the warp that the first of them falls to takes them all.
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
  int hkv, rows_per_block;
  int* status;
};

constexpr int kStoreFp8Threads = 256;

template <int D>
__global__ void __launch_bounds__(kStoreFp8Threads) store_fp8_kernel(const StoreFp8Params p) {
  constexpr int PIECES = D / 8;       // lanes that hold a row, eight values each
  constexpr int ROWS = 16 / PIECES;   // rows that a half of the warp takes at a time
  constexpr int HELD = kScaleGroup / ROWS;
  constexpr unsigned ALL = 0xffffffffu;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool is_v = lane >= 16;
  const int sub = (lane & 15) / PIECES, piece = lane % PIECES;
  const __nv_bfloat16* rows = is_v ? p.rows[1] : p.rows[0];
  const int64_t stride = is_v ? p.stride[1] : p.stride[0];
  unsigned char* cache = is_v ? p.cache[1] : p.cache[0];
  float* scales = is_v ? p.scale[1] : p.scale[0];

  pdl_wait();
  pdl_trigger();
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.rows_per_block;
  const int n_here = static_cast<int>(min(static_cast<int64_t>(p.rows_per_block), p.n - r0));
  auto slot_at = [&](int64_t r) -> int {  // -1: nothing is stored
    if (r < 0 || r >= p.n) return -1;
    const int s = p.slots[r];
    return s < p.num_slots ? max(s, -1) : -1;
  };
  const int slot = lane < n_here ? slot_at(r0 + lane) : -1;
  if (warp == 0 && lane < n_here && p.slots[r0 + lane] >= p.num_slots) atomicOr(p.status, NVLLM_STATUS_BAD_SLOT);
  const unsigned live = __ballot_sync(ALL, slot >= 0);
  if (!live) return;
  // the group of the last stored row before this block's
  int before = -1;
#pragma unroll 1
  for (int64_t r = r0 - 32; r > -32; r -= 32) {
    const int s = slot_at(r + lane);
    const unsigned m = __ballot_sync(ALL, s >= 0);
    if (m) {
      before = __shfl_sync(ALL, s, 31 - __clz(m)) / kScaleGroup;
      break;
    }
  }
  const int group = slot >= 0 ? slot / kScaleGroup : -1;
  const unsigned below = live & ((1u << lane) - 1);
  const int previous = __shfl_sync(ALL, group, below ? 31 - __clz(below) : lane);
  const unsigned leaders = __ballot_sync(ALL, slot >= 0 && group != (below ? previous : before));

#pragma unroll 1
  for (int u = warp; u < __popc(leaders) * p.hkv; u += warps) {
    const int head = u % p.hkv;
    unsigned left = leaders;
    for (int k = u / p.hkv; k > 0; --k) left &= left - 1;
    const int at = __ffs(left) - 1;
    const int g = __shfl_sync(ALL, group, at);
    const int64_t i = r0 + at;
    const __nv_bfloat16* src = rows + head * D + piece * 8;
    // Rows i + b, b < 32, of this group: bits b.  `ended`: a row of another group follows, or none.
    auto window = [&](int64_t from, int& s, bool& ended) {
      s = slot_at(from + lane);
      const unsigned same = __ballot_sync(ALL, s >= 0 && s / kScaleGroup == g);
      const unsigned other = __ballot_sync(ALL, s >= 0 && s / kScaleGroup != g);
      ended = other != 0 || from + 32 >= p.n;
      return other ? same & ((other & -other) - 1) : same;
    };
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
    auto load = [&](int64_t r) { return __ldg(reinterpret_cast<const uint4*>(src + r * stride)); };

    int s;
    bool ended;
    const unsigned run = window(i, s, ended);
    const bool held = ended && __popc(run) <= kScaleGroup;  // all rows of the group in registers
    int first = __reduce_min_sync(ALL, run >> lane & 1u ? s % kScaleGroup : kScaleGroup);
    uint4 x[HELD];
    uint32_t most = 0;
    auto fold = [&](const uint4& v) {
      most = max_finite2(max_finite2(max_finite2(max_finite2(most, v.x), v.y), v.z), v.w);
    };
    float* scale_at = scales + (static_cast<int64_t>(g / kGroups) * p.hkv + head) * kGroups + g % kGroups;
    float old = 0.f;
    if (held) {
      unsigned m = run;
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        const int b = next_rows(m);
        x[j] = b >= 0 ? load(i + b) : make_uint4(0, 0, 0, 0);
      }
      if (first > 0) old = *scale_at;
#pragma unroll
      for (int j = 0; j < HELD; ++j) fold(x[j]);
    } else {  // the same slots over and over
      int64_t from = i;
#pragma unroll 1
      while (true) {
        int s2;
        bool end2;
        unsigned m = window(from, s2, end2);
        first = min(first, __reduce_min_sync(ALL, m >> lane & 1u ? s2 % kScaleGroup : kScaleGroup));
#pragma unroll 1
        while (m) {
          const int b = next_rows(m);
          if (b >= 0) fold(load(from + b));
        }
        if (end2) break;
        from += 32;
      }
      if (first > 0) old = *scale_at;
    }
    most = max(most & 0xffffu, most >> 16);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(ALL, most, d));
    const int e = first > 0 ? max(exponent_for(most), exponent_of(old)) : exponent_for(most);
    const float now = power_of_two(e), inv = power_of_two(-e);
    if (first > 0 && now != old) {  // a half warp at most: no shuffles in here
      const float ratio = old * inv;
#pragma unroll 1
      for (int r = sub; r < first; r += ROWS) {
        uint2* c = reinterpret_cast<uint2*>(cache + ((static_cast<int64_t>(g) * kScaleGroup + r) * p.hkv + head) * D + piece * 8);
        const uint2 v = *c;
        *c = make_uint2(recode4(v.x, ratio), recode4(v.y, ratio));
      }
    }
    __syncwarp();
    auto store = [&](const uint4& v, int to) {
      *reinterpret_cast<uint2*>(cache + (static_cast<int64_t>(to) * p.hkv + head) * D + piece * 8) = encode8(v, inv);
    };
    // Rows in order, so that of two with the same slot the later one stays; of two at a time the first only where they differ.
    auto destination = [&](int sl, int b) {
      const int to = __shfl_sync(ALL, sl, max(b, 0));
      const int later = ROWS == 2 ? __shfl_down_sync(ALL, b >= 0 ? to : -1, PIECES) : -1;
      return b < 0 || (ROWS == 2 && sub == 0 && later == to) ? -1 : to;
    };
    if (held) {
      unsigned m = run;
#pragma unroll
      for (int j = 0; j < HELD; ++j) {
        const int to = destination(s, next_rows(m));
        if (to >= 0) store(x[j], to);
        __syncwarp();
      }
    } else {
      int64_t from = i;
#pragma unroll 1
      while (true) {
        int s2;
        bool end2;
        unsigned m = window(from, s2, end2);
#pragma unroll 1
        while (m) {
          const int b = next_rows(m);
          const int to = destination(s2, b);
          if (to >= 0) store(load(from + b), to);
          __syncwarp();
        }
        if (end2) break;
        from += 32;
      }
    }
    if ((lane & 15) == 0) *scale_at = now;
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
  p.rows_per_block = n_tokens <= 4096 ? 1 : kScaleGroup;
  const int64_t blocks = (n_tokens + p.rows_per_block - 1) / p.rows_per_block;
  if (blocks > 0x7fffffffLL) return fail(NVLLM_E_GEOMETRY, "store_kvcache_fp8: too many tokens for one launch");
  const int threads = 32 * (num_kv_heads < kStoreFp8Threads / 32 ? num_kv_heads : kStoreFp8Threads / 32);
  return launch_kernel("store_kvcache_fp8", head_dim == 128 ? store_fp8_kernel<128> : store_fp8_kernel<64>,
                       dim3(static_cast<unsigned>(blocks)), dim3(threads), 0, static_cast<cudaStream_t>(stream), p);
}
