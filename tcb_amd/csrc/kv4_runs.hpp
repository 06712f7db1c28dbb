// kv4_runs.hpp -- which tokens a workgroup of the 4-bit cache's row kernels takes together (kv4.hip; also compiled by a host compiler).
#pragma once

#include <cstdint>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define KV4_BOTH __host__ __device__ __forceinline__
#else
#define KV4_BOTH inline
#endif

namespace trhip {

// Token numbers are unsigned: there are up to 2^31 - 1, and a workgroup's next one, four times 65535 further, and the three behind a token must not
// wrap.
constexpr uint32_t kKv4Groups = 65535;  // at most, in a launch's second dimension
constexpr uint32_t kv4_next(uint32_t t0, uint32_t groups, uint32_t run) { return t0 + groups * run; }

// The token's slot and how many tokens the workgroup of token t takes: 4 where t is the first of four in a row from a multiple of four,
// 0 where an earlier workgroup takes it (or it has no slot). slots: an array, or what stands for one.
template <class Slots> KV4_BOTH int kv4_together(const Slots &slots, uint32_t tokens, int64_t places, uint32_t t, int64_t &slot) {
    slot = slots[t];
    if ((uint64_t)slot >= (uint64_t)places) return 0;
    const uint32_t at = (uint32_t)(slot & 3), first = t - at;
    if (at > t || first + 3 >= tokens) return 1;
    bool row = true;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) row = row && (int64_t)slots[first + i] == slot - at + i;
    return !row ? 1 : at == 0 ? 4 : 0;
}

}  // namespace trhip
