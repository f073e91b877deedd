// Grouped-query attention over a cache held in 4 bits (q4_cache.cuh).
#pragma once
#include "q4_cache.cuh"

namespace zk {

struct Q4Attend {
    Q4Cache cache;
    Q4Rotation turn;
    const float* q;            // rows q_ld apart
    const int* position;
    const int* filled;
    const float* weight_in;    // [kv_heads][slots]
    float* weight_out;         // or null
    float* out;                // [tokens][heads * head_dim]
    float* stats;              // workspace [tokens][heads][2]: a row's largest score and the sum of its exponentials
    uint32_t tokens, heads;
    size_t q_ld;
    float scale;
    int* error_word;
};

// A block's value at `lane`.
__device__ __forceinline__ float q4_value(const uint8_t* codes, const __half* scales, uint32_t h, uint32_t slot, uint32_t block, uint32_t lane, const Q4Cache& c) {
    const uint32_t byte = __ldcg(codes + q4_codes_at(h, slot, block, c.blocks, c.slots) + (lane & 15u));
    return (static_cast<float>(lane < 16 ? byte & 15u : byte >> 4) - 8.0f) * __half2float(__ldcg(scales + q4_scale_at(h, slot, block, c.blocks, c.slots)));
}
template <int kBlocks>
__device__ __forceinline__ float q4_score(const float (&q)[kBlocks], uint32_t h, uint32_t slot, uint32_t lane, const Q4Attend& p) {
    float s = 0.0f;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) s = fmaf(q[b], q4_value(p.cache.k_codes, p.cache.k_scales, h, slot, b, lane, p.cache), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s * p.scale;
}

// A CTA of eight warps takes a row (token t, query head); a warp every eighth slot.
template <int kBlocks>
__global__ void __launch_bounds__(256) q4_attend_kernel(const __grid_constant__ Q4Attend p) {
    __shared__ float share_out[8][kBlocks * 32], share_max[8], share_sum[8];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, t = blockIdx.x, head = blockIdx.y, h = head / (p.heads / p.cache.kv_heads);
    pdl_launch_dependents();
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;
    float q[kBlocks], acc[kBlocks] = {};
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) q[b] = q4_rotated(p.q + t * p.q_ld + static_cast<size_t>(head) * kBlocks * 32, b * 32 + lane, p.turn, static_cast<size_t>(position) + t);
    float m = -INFINITY, l = 0.0f;
    for (uint32_t slot = warp; slot <= static_cast<uint32_t>(filled) + t; slot += 8) {
        const float s = q4_score<kBlocks>(q, h, slot, lane, p), top = fmaxf(m, s);
        const float corr = m == -INFINITY ? 0.0f : expf(m - top), e = expf(s - top);
        l = l * corr + e;
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) acc[b] = acc[b] * corr + e * q4_value(p.cache.v_codes, p.cache.v_scales, h, slot, b, lane, p.cache);
        m = top;
    }
    for (int b = 0; b < kBlocks; ++b) share_out[warp][b * 32 + lane] = acc[b];
    if (lane == 0) { share_max[warp] = m; share_sum[warp] = l; }
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < 8; ++w) top = fmaxf(top, share_max[w]);
    float factor[8];
    for (int w = 0; w < 8; ++w) {
        factor[w] = share_max[w] == -INFINITY ? 0.0f : expf(share_max[w] - top);
        sum += factor[w] * share_sum[w];
    }
    if (threadIdx.x == 0) {
        if (!(sum > 0.0f) || !(sum < INFINITY)) atomicExch(p.error_word, kErrNonFinite);
        p.stats[(static_cast<size_t>(t) * p.heads + head) * 2] = top;
        p.stats[(static_cast<size_t>(t) * p.heads + head) * 2 + 1] = sum;
    }
    for (uint32_t e = threadIdx.x; e < kBlocks * 32; e += 256) {
        float o = 0.0f;
        for (int w = 0; w < 8; ++w) o += factor[w] * share_out[w][e];
        p.out[(static_cast<size_t>(t) * p.heads + head) * kBlocks * 32 + e] = o / sum;
    }
}

// A warp takes a slot: the weights its group's rows gave it.
template <int kBlocks>
__global__ void __launch_bounds__(256) q4_received_kernel(const __grid_constant__ Q4Attend p) {
    const uint32_t lane = threadIdx.x & 31u, slot = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y, group = p.heads / p.cache.kv_heads;
    pdl_launch_dependents();
    pdl_wait();
    const int filled = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions) || slot >= filled + p.tokens) return;
    float sum = 0.0f;
    for (uint32_t t = slot < static_cast<uint32_t>(filled) ? 0 : slot - filled; t < p.tokens; ++t)
        for (uint32_t j = 0; j < group; ++j) {
            const uint32_t head = h * group + j;
            float q[kBlocks];
            for (int b = 0; b < kBlocks; ++b) q[b] = q4_rotated(p.q + t * p.q_ld + static_cast<size_t>(head) * kBlocks * 32, b * 32 + lane, p.turn, static_cast<size_t>(position) + t);
            const float* stats = p.stats + (static_cast<size_t>(t) * p.heads + head) * 2;
            sum += expf(q4_score<kBlocks>(q, h, slot, lane, p) - __ldcg(stats)) / __ldcg(stats + 1);
        }
    if (lane == 0) {
        const size_t at = static_cast<size_t>(h) * p.cache.slots + slot;
        p.weight_out[at] = sum + (slot < static_cast<uint32_t>(filled) ? p.weight_in[at] : 0.0f);
    }
}

}  // namespace zk
