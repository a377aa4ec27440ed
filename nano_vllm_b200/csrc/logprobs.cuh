// Running softmax statistics of a row with its entropy, shared by the kernels that score tokens.
#pragma once

#include <cfloat>

#include "common.cuh"

namespace nvllm {

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 1 / T of a row; a temperature that is not above 0, or none, counts as 1.  Beyond 1e30 it counts as 1e30: every logit up to 1e22 is
// uniform there already, and a masked one's difference, -3e38 at the least, still has no weight.  Below 1e-38 it counts as 1e-38, whose
// inverse is finite; a comparison, as this is compiled, would take subnormal ones for 0.
__device__ __forceinline__ float lp_inverse(const float* temperatures, int64_t row) {
  const float t = temperatures ? temperatures[row] : 1.f;
  const int bits = __float_as_int(t);
  return bits > 0 && bits <= 0x7f800000 ? fminf(fmaxf(__frcp_rn(t), 1e-30f), 1e38f) : 1.f;
}

// Maximum m (no less than the smallest finite number), s = sum exp2(c (x - m)), t = sum exp2(c (x - m)) (x - m).
struct LpSums {
  float m, s, t;
  // Differences of -infinity: no weight, and 0 and not NaN times that.
  static __device__ __forceinline__ float diff(float a, float m) { return max_nan(a - m, -3e38f); }
  __device__ __forceinline__ void rescale(float to, float c) {
    const float d = diff(m, to), f = fast_exp2(d * c);
    s *= f;
    t = fmaf(s, d, f * t);  // s first: times d it may not overflow
    m = to;
  }
  __device__ __forceinline__ void join(float m2, float s2, float t2, float c) {
    LpSums o{m2, s2, t2};
    const float to = fmaxf(m, m2);
    rescale(to, c);
    o.rescale(to, c);
    s += o.s;
    t += o.t;
  }
  // ln of the sum, which is 1 or more, 0 (nothing but -infinity) or NaN, to about 2^-23 of itself: near 1, where one token has nearly
  // all of it, as well.  s = 2^e f with f within sqrt(1/2) and sqrt(2); ln f = 2 artanh z, z = (f - 1) / (f + 1), |z| < 0.172: the
  // series ends before 2 z^11 / 11 < 8e-10.  (log() in 64 bits takes 1 us at the end of every row.)
  __device__ __forceinline__ float log_z() const {
    if (!(s > 0.f)) return s == 0.f ? -INFINITY : NAN;
    const int e = (__float_as_int(s) - 0x3f3504f3) >> 23;  // sqrt(1/2)
    const float f = __int_as_float(__float_as_int(s) - (e << 23)), z = __fdiv_rn(f - 1.f, f + 1.f), z2 = z * z;
    const float series = fmaf(z2, fmaf(z2, fmaf(z2, fmaf(z2, 1.f / 9, 1.f / 7), 1.f / 5), 1.f / 3), 1.f);
    return fmaf(static_cast<float>(e), 0.693147182f, 2.f * z * series);
  }
  __device__ __forceinline__ void results(int64_t row, int64_t token, float given, float inv_t, float log_z, int vocab, float* logprobs,
                                          float* entropy, int* status) const {
    float lp = 0.f;
    if (token >= vocab) {
      lp = NAN;
      atomicOr(status, NVLLM_STATUS_BAD_TOKEN);
    } else if (token >= 0) {
      lp = (given - m) * inv_t - log_z;
    }
    logprobs[row] = lp;
    entropy[row] = log_z - inv_t * __fdiv_rn(t, s);
  }
};

}  // namespace nvllm
