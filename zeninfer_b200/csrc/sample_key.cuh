// What the sampler and the check of drafted tokens share.
#pragma once
#include <cstdint>

namespace zk {

constexpr uint32_t kSampleMaxCandidates = 1024;

// Order-preserving key of a finite float (larger float, larger key); 0 for a non-finite one (never a candidate).
__device__ __forceinline__ uint32_t sample_key(float v) {
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7f800000u) == 0x7f800000u) return 0u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

}  // namespace zk
