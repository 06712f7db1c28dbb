// rope.hpp -- what of the rotary positions needs no device: the series of sine and cosine (for tests also in 64 bits), the sizes of launches.
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define ROPE_BOTH __host__ __device__ __forceinline__
#else
#define ROPE_BOTH inline
#endif

namespace trhip {

ROPE_BOTH float rope_fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
ROPE_BOTH double rope_fma(double a, double b, double c) { return __builtin_fma(a, b, c); }

// Taylor series on |x| <= pi / 4, z = x^2; they leave out x^11 / 11! and x^12 / 12!, 2^-29 at most and 2^-33.
template <class T> ROPE_BOTH T rope_sin(T x, T z) {
    const T y = rope_fma(z, rope_fma(z, rope_fma(z, T(2.7557319e-6), T(-1.98412698e-4)), T(8.33333333e-3)), T(-1.66666667e-1));
    return rope_fma(z * x, y, x);
}
template <class T> ROPE_BOTH T rope_cos(T z) {
    const T y = rope_fma(z, rope_fma(z, rope_fma(z, T(-2.7557319e-7), T(2.48015873e-5)), T(-1.38888889e-3)), T(4.16666667e-2));
    return rope_fma(z, rope_fma(z, y, T(-0.5)), T(1));
}

// A launch of the first of `left` tokens, `each` (one or four) a workgroup. Workgroups times threads has to stay below 2^32, so a launch has
// 2^23 tokens at most, a multiple of four, and 2^31 threads.
constexpr int kRopeThreads = 256;
constexpr int64_t kRopeTokens = (int64_t)1 << 23;
struct RopeLaunch {
    int tokens;
    unsigned groups;
};
inline RopeLaunch rope_launch(int64_t left, int each) {
    const int tokens = (int)(left < kRopeTokens ? left : kRopeTokens);
    return {tokens, (unsigned)((tokens + each - 1) / each)};
}

}  // namespace trhip
