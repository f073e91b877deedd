// Attention of a block of many rows over a cache held in 4 bits, heads of 64 or 128 values, on the tensor cores (tcgen05).
//
// The formulas and the bookkeeping are q4_attention.cuh's: queries and weights enter as two f16 numbers each, keys and values are exact.  What differs is where a
// block's scale goes.  Here it goes into the operand: d (c - 8) is a number of fifteen bits, exactly the sum of two f16 numbers (the rounded product and
// its remainder, a multiplication and a multiply-add of halves), so a product is three products of f16 numbers (the fourth is below 2^-22 of it), and nothing has to be
// done per block and score.  A tile's scales are multiplied by the power of two that brings the largest below 2^9, so that both parts keep their bits
// whatever the model's magnitudes are.  The dimensions of the operands stand in the order in which the nibbles are unpacked.
//
// A CTA takes 128 rows (a row: a token times a query head of the kv head, any group) and walks its run of slots 64 at a time.  24 warps:
//   16 rows      a thread has a quarter of a row: 16 scores from TMEM, mask, running maximum (of the quarters), exponentials, the weights' two parts back to
//                TMEM, from where the tensor cores read them (as they do the queries); then out = out * factor + O' of the tile before, in fp32 registers
//   3 + 4        unpack keys and values (bulk copies bring the tiles into a ring, two ahead) into the operands' 128-byte swizzle, two buffers each, a slot's block a
//                thread: to the tensor cores keys are a matrix with the summed index in its rows, values one with it in its columns, so neither is transposed
//   1 issues     S = Q K^T into three accumulators in turn (a product waits for the sum that it adds to, and the tensor cores cut a sum at every 16 columns), O' = P V;
//                corrections first
// The scores of tile j + 1 are formed while tile j is exponentiated.
//
// What bounds it: the chain of a row's warps (scores out of TMEM, maximum of the quarters, exponentials, split, weights into TMEM, output sum), some 4000 cycles a tile, beside which
// the matrix instructions take 2000 and unpacking, shared by all rows of the CTA, 3000.  512 tokens (2048 rows of 8 kv heads of 128): 33 us into an empty cache with the append,
// 346 us into 7680 slots with the append and the weights received.  Measured on the way there, the last case: values unpacked transposed 1000 us of attention alone, as the
// transposed operand 420, four threads a row instead of two 350, elect.sync 230.
//
// A scale that is not finite counts as zero in the operands and is remembered by its slot: the rows that see it are NaN (all of them for a key's, the
// block's dimensions for a value's), and the others know nothing of it.
#pragma once
#include "attention_tc.cuh"
#include "q4_attention.cuh"

namespace zk {

constexpr uint32_t kQpRows = 128, kQpKeys = 64, kQpThreads = 24 * 32, kQpKeyWarp = 16, kQpValueWarp = 19, kQpIssueWarp = 23;      // first warps of the roles
template <int kBlocks> constexpr uint32_t kQpQPlane = kQpRows * kBlocks * 64;      // bytes
template <int kBlocks> constexpr uint32_t kQpKPlane = kQpKeys * kBlocks * 64;      // of keys, of values
constexpr int kQpStages = 3;                 // tiles as they are in the cache, ahead of the warps that unpack them
template <int kBlocks> constexpr uint32_t kQpRaw = kQpKeys * kBlocks * 36;
template <int kBlocks> constexpr uint32_t q4_prompt_smem() { return 1024 + 2 * kQpQPlane<kBlocks> + 8 * kQpKPlane<kBlocks> + kQpStages * kQpRaw<kBlocks>; }
// TMEM columns: three shares of the scores; the weights' parts; O'; the queries' parts
constexpr uint32_t kQpScores = 0, kQpShares = 3, kQpP = 192, kQpOut = 256, kQpQ = 384, kQpColumns = 512;

// Instruction descriptor, kind::f16: f16 x f16 -> fp32, dense, A K-major, B K-major or (across) MN-major.
__host__ __device__ constexpr uint32_t umma_idesc_f16(uint32_t m, uint32_t n, bool across = false) { return (1u << 4) | (across ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((m >> 4) << 24); }
// Shared-memory descriptor of an MN-major operand with the 128-byte swizzle: rows of 64 columns (128 bytes), one for each index that is summed over, eight of them a group of
// 1024 bytes; the next 64 columns begin `apart` bytes on.
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t smem_addr, uint32_t apart) {
    return (umma_desc_k_sw128(smem_addr) & ~(static_cast<uint64_t>(0x3fff) << 16)) | (static_cast<uint64_t>(apart >> 4) << 16);
}

__device__ __forceinline__ uint32_t f16x2_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t f16x2_rest(uint32_t a, uint32_t b, uint32_t product) {      // a * b - product
    uint32_t r;
    asm("{ .reg .b32 n; neg.f16x2 n, %3; fma.rn.f16x2 %0, %1, %2, n; }" : "=r"(r) : "r"(a), "r"(b), "r"(product));
    return r;
}
// One lane of a warp that is together, the same one every time.  What it guards is known to run in one thread, so that the operands of a matrix instruction stay in uniform
// registers: 24 of them are issued in 760 cycles, behind `lane == 0` in 1280, and beside warps that keep the scheduler busy in 1900 after 13000.
__device__ __forceinline__ bool elected() {
    uint32_t r;
    asm volatile("{ .reg .pred e; elect.sync _|e, 0xffffffff; selp.u32 %0, 1, 0, e; }" : "=r"(r));
    return r != 0;
}
// The power of two for a tile whose largest scale has these bits: times 2^shift it is below 2^9.
__device__ __forceinline__ int q4_shift(uint32_t top) { return 23 - static_cast<int>(top >> 10); }
__device__ __forceinline__ bool q4_finite(uint32_t half_bits) { return (half_bits & 0x7c00u) != 0x7c00u; }

// The largest magnitude among the finite scales of the first `slots` of kSlots slots, as f16 bits: every lane of a warp.  bad(slot, block) is called for the others.
template <int kBlocks, uint32_t kSlots, typename Bad>
__device__ __forceinline__ uint32_t q4_largest_scale(const __half* scales, uint32_t slots, uint32_t lane, Bad bad) {
    uint32_t both = 0;                                        // two maxima side by side
#pragma unroll
    for (uint32_t at = 0; at < kSlots * kBlocks / 8; at += 32) {      // eight scales a lane: 8 / kBlocks slots
        const uint32_t first = (at + lane) * 8 / kBlocks;
        if (first >= min(slots, kSlots)) continue;
        const uint4 eight = reinterpret_cast<const uint4*>(scales)[at + lane];
        uint32_t w[4] = {eight.x, eight.y, eight.z, eight.w};
        if (slots < kSlots) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (first + j / kBlocks >= slots) w[j / 2] &= j % 2 ? 0x0000ffffu : 0xffff0000u;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) both = __vmaxu2(both, w[j] & 0x7fff7fffu);
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, max(both & 0xffffu, both >> 16));
    if (q4_finite(top)) return top;
    top = 0;
#pragma unroll 1
    for (uint32_t i = lane; i < min(slots, kSlots) * kBlocks; i += 32) {
        const uint32_t bits = __half_as_ushort(scales[i]) & 0x7fffu;
        if (q4_finite(bits)) top = max(top, bits);
        else bad(i / kBlocks, i % kBlocks);
    }
    return __reduce_max_sync(0xffffffffu, top);
}

// Eight dimensions of a row of queries in the scores' order, 4j .. 4j+3 and 16+4j .. 16+4j+3 of a block, as they are unpacked from a word of codes.
__device__ __forceinline__ void q4_split_queries(const float (&x)[8], float up, uint4& upper, uint4& lower) {
    uint32_t u[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = (i & 1) * 4 + (i >> 1);            // {4j, 4j+2}, {16+4j, 16+4j+2}, {4j+1, 4j+3}, {17+4j, 19+4j}
        const float a = x[at] * up, b = x[at + 2] * up, ua = upper_digit(a), ub = upper_digit(b);
        u[i] = pack_f16(ua, ub);
        l[i] = pack_f16(a - ua, b - ub);
    }
    upper = make_uint4(u[0], u[1], u[2], u[3]);
    lower = make_uint4(l[0], l[1], l[2], l[3]);
}
// A word of codes (eight dimensions) times a scale: the operand's sixteen bytes in both planes.
__device__ __forceinline__ void q4_split_codes(uint32_t w, uint32_t d2, uint4& upper, uint4& lower) {
    const uint32_t x = w >> 8, c[4] = {signed_low(w), signed_high(w), signed_low(x), signed_high(x)};
    uint32_t u[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u[i] = f16x2_mul(c[i], d2);
        l[i] = f16x2_rest(c[i], d2, u[i]);
    }
    upper = make_uint4(u[0], u[1], u[2], u[3]);
    lower = make_uint4(l[0], l[1], l[2], l[3]);
}

// The codes of kSlots slots, as the cache holds them, times their scales, 2^shift as large, into both planes: rows of 64 dimensions a slot.  Scales that are not finite
// count as zero, and so do the slots from `slots` on, of which nothing is read.  kThreads threads, the id-th of them here.
template <int kBlocks, uint32_t kSlots, uint32_t kThreads>
__device__ __forceinline__ void q4_unpack_tile(const uint8_t* codes, const __half* scales, uint32_t slots, int shift, uint8_t* to, uint32_t id) {
    constexpr uint32_t kItems = kSlots * kBlocks, kEach = (kItems + kThreads - 1) / kThreads, kPlane = kSlots * kBlocks * 64, kHalves = kBlocks / 2;
    const float up = power_of_two(shift);
#pragma unroll
    for (uint32_t i = 0; i < kEach; ++i) {
        const uint32_t item = id + kThreads * i, r = item % kSlots, block = item / kSlots;
        if (kItems % kThreads && item >= kItems) break;       // a whole warp
        uint4 four = make_uint4(0, 0, 0, 0);
        uint32_t bits = 0;
        if (r < slots) {
            four = *reinterpret_cast<const uint4*>(codes + (((r >> 3) * kBlocks + block) * 8 + (r & 7u)) * 16);
            bits = __half_as_ushort(scales[r * kBlocks + block]);
        }
        if (!q4_finite(bits)) bits = 0;
        const float d = __half2float(__ushort_as_half(static_cast<unsigned short>(bits))) * up;
        const uint32_t d2 = pack_f16(d, d), w[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
        for (uint32_t word = 0; word < 4; ++word) {
            uint4 upper, lower;
            q4_split_codes(w[word], d2, upper, lower);
            const uint32_t at = (block / 2) * (kPlane / kHalves) + r * 128 + ((((block & 1) * 4 + word) ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(to + at) = upper;
            *reinterpret_cast<uint4*>(to + kPlane + at) = lower;
        }
    }
}

// grid = (splits, tiles of 128 rows, kv_heads); the rows that see most slots come first.
template <int kBlocks>
__global__ void __launch_bounds__(kQpThreads, 1) q4_prompt_kernel(const __grid_constant__ Q4Attend p) {
    constexpr uint32_t kDim = kBlocks * 32, kHalves = kBlocks / 2, kQPlane = kQpQPlane<kBlocks>, kKPlane = kQpKPlane<kBlocks>;
    extern __shared__ uint8_t qp_smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(qp_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* const q_smem = smem;                             // [plane][64 dimensions][128 rows][128 bytes]
    uint8_t* const k_smem = q_smem + 2 * kQPlane;             // [buffer][plane][64 dimensions][64 slots][128 bytes]
    uint8_t* const v_smem = k_smem + 4 * kKPlane;             // the same
    uint8_t* const raw_smem = v_smem + 4 * kKPlane;           // [stage]: codes of keys and of values, scales of keys and of values
    __shared__ float row_factor[kQpRows], top[2][4][kQpRows], sum[4][kQpRows];
    __shared__ uint64_t raw_full[kQpStages], raw_free[kQpStages], k_full[2], k_free[2], v_full[2], v_free[2], q_full, s_full, s_empty, p_full, o_full, o_empty;
    __shared__ float k_unit[4], v_unit[4];                    // what a tile's operands are to be multiplied by: the rows read the last but one while the next is stored
    __shared__ uint32_t tmem_slot, bad_key, bad_value[kBlocks];      // the first slots whose scales are not finite
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, h = blockIdx.z, rows = p.tokens * p.group;
    const uint32_t first_row = (gridDim.y - 1 - blockIdx.y) * kQpRows, real_rows = min(kQpRows, rows - first_row);
    if (threadIdx.x == 0) {
        for (int b = 0; b < kQpStages; ++b) { mbar_init(&raw_full[b], 1); mbar_init(&raw_free[b], kQpIssueWarp - kQpKeyWarp); }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&k_full[b], kQpValueWarp - kQpKeyWarp); mbar_init(&v_full[b], kQpIssueWarp - kQpValueWarp);
            mbar_init(&k_free[b], 1); mbar_init(&v_free[b], 1);
        }
        mbar_init(&q_full, kQpKeyWarp); mbar_init(&s_full, 1); mbar_init(&s_empty, kQpKeyWarp); mbar_init(&p_full, kQpKeyWarp); mbar_init(&o_full, 1); mbar_init(&o_empty, kQpKeyWarp);
        mbar_fence_init();
        bad_key = 0xffffffffu;
        for (int b = 0; b < kBlocks; ++b) bad_value[b] = 0xffffffffu;
    }
    pdl_launch_dependents();
    pdl_wait();
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;      // the append has said so
    const uint32_t filled = filled_in, seen = filled + (first_row + real_rows - 1) / p.group + 1;                 // slots of the last token
    const Q4Runs runs = q4_runs(seen, p.splits, 1, kQpKeys);
    const uint32_t begin = blockIdx.x * runs.per, end = min(runs.tiles, begin + runs.per);
    if (begin >= end) return;                                                            // nobody counts on this run
    if (warp == kQpIssueWarp) tmem_alloc(&tmem_slot, kQpColumns);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    constexpr uint32_t kCodes = kQpKeys * kBlocks * 16, kScales = kQpKeys * kBlocks * 2;
    auto bring = [&](uint32_t tile, int stage) {              // the last tile may have half of its slots beyond the cache's end
        const uint32_t slots = min(kQpKeys, p.cache.slots - tile * kQpKeys);
        const size_t slot = static_cast<size_t>(h) * p.cache.slots + static_cast<size_t>(tile) * kQpKeys;
        uint8_t* to = raw_smem + stage * kQpRaw<kBlocks>;
        mbar_arrive_expect_tx(&raw_full[stage], slots * kBlocks * 36);
        bulk_g2s(to, p.cache.k_codes + slot * (kBlocks * 16), slots * kBlocks * 16, &raw_full[stage]);
        bulk_g2s(to + kCodes, p.cache.v_codes + slot * (kBlocks * 16), slots * kBlocks * 16, &raw_full[stage]);
        bulk_g2s(to + 2 * kCodes, p.cache.k_scales + slot * kBlocks, slots * kBlocks * 2, &raw_full[stage]);
        bulk_g2s(to + 2 * kCodes + kScales, p.cache.v_scales + slot * kBlocks, slots * kBlocks * 2, &raw_full[stage]);
    };
    if (warp < kQpKeyWarp) {      // Q, while the other warps begin with the tiles: a thread takes eight dimensions of several rows, neighbouring threads a row's, all asked for first
        constexpr uint32_t kChunks = kDim / 8, kRowThreads = kQpKeyWarp * 32, kEach = kQpRows * kChunks / kRowThreads;
        const uint32_t chunk = threadIdx.x % kChunks, dim = chunk / 4 * 32 + chunk % 4 * 4;
        float x[kEach][8];
        auto ask = [&](auto turn) {                           // which way they turn is decided once, so that no row's loads wait for another's
            constexpr int kTurn = decltype(turn)::value;
#pragma unroll
            for (uint32_t i = 0; i < kEach; ++i) {
                const uint32_t r = threadIdx.x / kChunks + i * (kRowThreads / kChunks), row = first_row + min(r, real_rows - 1), token = row / p.group;
                const float* from = p.q + token * p.q_ld + static_cast<size_t>(h * p.group + row % p.group) * kDim;
                const size_t turned = static_cast<size_t>(position) + token;
                if constexpr (kTurn < 3) q4_rotated_fours<kTurn>(x[i], from, dim, p.turn, turned);
                else q4_rotated_eight(x[i], from, dim, p.turn, turned, false);
            }
        };
        if (!q4_rotates_fours(p.q, p.q_ld, kDim, p.turn)) ask(std::integral_constant<int, 3>{});
        else if (!p.turn.pairs) ask(std::integral_constant<int, 0>{});
        else if (p.turn.adjacent) ask(std::integral_constant<int, 1>{});
        else ask(std::integral_constant<int, 2>{});
#pragma unroll
        for (uint32_t i = 0; i < kEach; ++i) {
            const uint32_t r = threadIdx.x / kChunks + i * (kRowThreads / kChunks);
            float most = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (r >= real_rows) x[i][e] = 0.0f;
                most = fmaxf(most, fabsf(x[i][e]));
            }
#pragma unroll
            for (uint32_t o = kChunks / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int e = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -114);
            uint4 upper, lower;
            q4_split_queries(x[i], p.scale < 0.0f ? -power_of_two(13 - e) : power_of_two(13 - e), upper, lower);
            const uint32_t at = (chunk / 8) * (kQPlane / kHalves) + r * 128 + (((chunk % 8) ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(q_smem + at) = upper;
            *reinterpret_cast<uint4*>(q_smem + kQPlane + at) = lower;
            if (chunk == 0) row_factor[r] = q4_row_factor(p.scale, e);
            // the same for the launch that adds up what the slots received
            if (p.queries && blockIdx.x == 0) {
                uint8_t* to = reinterpret_cast<uint8_t*>(p.queries) + (static_cast<size_t>(h) * gridDim.y + first_row / kQpRows) * 2 * kQPlane + at;
                *reinterpret_cast<uint4*>(to) = upper;
                *reinterpret_cast<uint4*>(to + kQPlane) = lower;
                if (chunk == 0) p.factors[static_cast<size_t>(h) * gridDim.y * kQpRows + first_row + r] = row_factor[r];
            }
        }
        // and into TMEM, half a row's part a thread: the products then read keys only from shared memory
        asm volatile("barrier.sync 9, %0;" ::"n"(kQpKeyWarp * 32) : "memory");
        const uint32_t r = (warp & 3u) * 32 + lane, plane = warp >> 3, c0 = (warp >> 2 & 1u) * (kDim / 32);
#pragma unroll
        for (uint32_t c = 0; c < kDim / 32; ++c) {
            uint32_t both[8];
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t chunk = 2 * (c0 + c) + i;
                const uint4 its = *reinterpret_cast<const uint4*>(q_smem + plane * kQPlane + (chunk / 8) * (kQPlane / kHalves) + r * 128 + (((chunk % 8) ^ (r & 7)) << 4));
                both[4 * i] = its.x; both[4 * i + 1] = its.y; both[4 * i + 2] = its.z; both[4 * i + 3] = its.w;
            }
            tmem_st_32x8(tmem + kQpQ + plane * (kDim / 2) + 8 * (c0 + c) + (((warp & 3u) * 32) << 16), both);
        }
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full);
    }
    auto gave_up = [&](int code) { if (lane == 0) atomicExch(p.error_word, code); };

    // A wait that runs out ends its role's loop, and the others' follow.
    if (warp < kQpKeyWarp) {                                  // rows
        const uint32_t quad = warp & 3, quarter = warp >> 2, r = quad * 32 + lane, row = first_row + r, lane_base = (quad * 32) << 16;
        const bool live = r < real_rows, any_live = quad * 32 < real_rows;      // warps without rows arrive where the others do, and leave TMEM as it is
        const uint32_t last_seen = live ? filled + row / p.group : 0xffffffffu;          // rows that are none: whatever comes, they write nothing
        constexpr int kMine = kQpKeys / 4, kOut = kDim / 4;
        const float factor = row_factor[r];
        // the four warps of a row meet; true where one of them has given up
        auto meet = [&](bool failed) {
            uint32_t any;
            asm volatile(
                "{ .reg .pred p, q; setp.ne.u32 q, %3, 0; barrier.red.or.pred p, %1, %2, q; selp.u32 %0, 1, 0, p; }"
                : "=r"(any) : "r"(quad + 1), "r"(128u), "r"(static_cast<uint32_t>(failed)) : "memory");
            return any != 0;
        };
        constexpr float kFull = 14.0f;                        // a weight of 1 is 2^14: its parts are f16's normal numbers over 2^20 and more
        float acc[kOut], m = -INFINITY, l = 0.0f, shrink = 0.0f;
#pragma unroll
        for (int i = 0; i < kOut; ++i) acc[i] = 0.0f;
        auto take_output = [&](float by) {                    // acc = acc * shrink + O'
            uint32_t v[kOut / 16][16];
#pragma unroll
            for (int b = 0; b < kOut / 16; ++b) tmem_ld_32x16(tmem + kQpOut + quarter * kOut + 16 * b + lane_base, v[b]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < kOut; ++i) acc[i] = fmaf(__uint_as_float(v[i / 16][i % 16]), by, acc[i] * shrink);
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty);
        };
        bool ok = true;
        uint32_t j = 0;
        for (uint32_t tile = begin; tile < end; ++tile, ++j) {
            ok = ok && warp_waited(&s_full, j & 1);
            float s[kMine], most = -INFINITY, by = 0.0f;
            if (!any_live) {
                if (ok && j > 0) ok = warp_waited(&o_full, (j - 1) & 1);
                if (!ok) break;
                if (lane == 0) {
                    mbar_arrive(&s_empty);
                    mbar_arrive(&p_full);
                    if (j > 0) mbar_arrive(&o_empty);
                }
                continue;
            }
            if (ok) {
                tc_fence_after_sync();
#pragma unroll
                for (int c = 0; c < kMine / 8; ++c) {
                    uint32_t part[3][8];
#pragma unroll
                    for (int i = 0; i < 3; ++i) tmem_ld_32x8(tmem + kQpScores + i * kQpKeys + quarter * kMine + 8 * c + lane_base, part[i]);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[8 * c + i] = (__uint_as_float(part[0][i]) + __uint_as_float(part[1][i])) + __uint_as_float(part[2][i]);
                }
                by = fmaxf(factor * k_unit[j & 3], kQ4LeastFactor);      // the unit of a tile of tiny scales, 2^-23, may take the least factor to zero
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&s_empty);
                const uint32_t first = tile * kQpKeys + quarter * kMine;
                if (!__all_sync(0xffffffffu, first + kMine - 1 <= last_seen)) {
#pragma unroll
                    for (int i = 0; i < kMine; ++i) if (first + i > last_seen) s[i] = -INFINITY;
                }
                float part[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kMine; ++i) part[i & 3] = fmaxf(part[i & 3], s[i]);
                most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * by;
                top[j & 1][quarter][r] = most;
                if (p.scores && live) {
                    float4* to = reinterpret_cast<float4*>(p.scores + (static_cast<size_t>(h) * rows + row) * p.cache.slots + first);
#pragma unroll
                    for (int i = 0; i < kMine / 4; ++i) if (first + 4 * i < p.cache.slots) to[i] = make_float4(s[4 * i] * by, s[4 * i + 1] * by, s[4 * i + 2] * by, s[4 * i + 3] * by);
                }
            }
            if (meet(!ok)) { ok = false; break; }
            most = fmaxf(fmaxf(fmaxf(top[j & 1][0][r], top[j & 1][1][r]), fmaxf(top[j & 1][2][r], top[j & 1][3][r])), m);
            most = ceilf(most);                               // a whole number: neither taking it off nor 2 to it is rounded
            const float from = most == -INFINITY ? kFull : kFull - most, f = exp2_fast(m - (kFull - from));          // exp2(-inf) = 0 on the first slots
            m = most;
            float part[4] = {};
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                s[i] = exp2_fast(fmaf(s[i], by, from));
                part[i & 3] += s[i];
            }
            l = l * f + ((part[0] + part[1]) + (part[2] + part[3]));
            if (j > 0) ok = warp_waited(&o_full, (j - 1) & 1);                  // the tile before: its output is formed, and P's place free
            if (ok) {
                tc_fence_after_sync();
                uint32_t upper[8], lower[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float a = s[2 * i], b = s[2 * i + 1], ua = upper_digit(a), ub = upper_digit(b);
                    upper[i] = pack_f16(ua, ub);
                    lower[i] = pack_f16(a - ua, b - ub);
                }
                tmem_st_32x8(tmem + kQpP + 8 * quarter + lane_base, upper);
                tmem_st_32x8(tmem + kQpP + 32 + 8 * quarter + lane_base, lower);
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full);
                if (j > 0) take_output(v_unit[(j - 1) & 3]);
            }
            shrink = f;
        }
        if (ok) ok = warp_waited(&o_full, (j - 1) & 1);
        if (ok && any_live) { tc_fence_after_sync(); take_output(v_unit[(j - 1) & 3]); }
        sum[quarter][r] = l;
        if (meet(!ok)) {
            gave_up(kErrTmemWaitTimeout);
        } else if (live) {
            l = ((sum[0][r] + sum[1][r]) + (sum[2][r] + sum[3][r])) * (1.0f / 16384.0f);
            if (last_seen >= bad_key) l = NAN;
            const bool alone = p.splits == 1;
            const float inv = alone ? 1.0f / l : 1.0f;
            const uint32_t token = row / p.group, head = h * p.group + row % p.group;
            const size_t part = (static_cast<size_t>(h) * p.splits + blockIdx.x) * rows + row;
            float* const to = alone ? p.out + (static_cast<size_t>(token) * p.heads + head) * kDim : p.part_out + part * kDim;
            const bool fours = reinterpret_cast<uintptr_t>(to) % 16 == 0;
#pragma unroll
            for (int w = 0; w < kOut / 8; ++w) {              // a word's eight dimensions, where the nibbles are unpacked to: 4w .. 4w + 3 and 16 more
                const uint32_t word = quarter * (kOut / 8) + w, block = word / 4;
                const float by = last_seen >= bad_value[block] ? NAN : inv;
#pragma unroll
                for (int high = 0; high < 2; ++high) {
                    const int at = 8 * w + 2 * high;
                    const float4 o = make_float4(acc[at] * by, acc[at + 4] * by, acc[at + 1] * by, acc[at + 5] * by);
                    float* const here = to + block * 32 + high * 16 + word % 4 * 4;
                    if (fours) *reinterpret_cast<float4*>(here) = o;
                    else { here[0] = o.x; here[1] = o.y; here[2] = o.z; here[3] = o.w; }
                }
            }
            if (quarter == 0) {
                if (alone) {
                    if (!(l > 0.0f) || !(l < INFINITY)) atomicExch(p.error_word, kErrNonFinite);
                    if (p.stats) p.stats[static_cast<size_t>(h) * rows + row] = m + log2f(l);
                }
                if (!alone || p.scores) reinterpret_cast<float2*>(p.part_stats)[part] = make_float2(m, l);
            }
        }
    } else if (warp < kQpValueWarp) {                         // keys: a thread takes blocks of a slot
        constexpr uint32_t kId = (kQpValueWarp - kQpKeyWarp) * 32;
        const uint32_t id = threadIdx.x - kQpKeyWarp * 32, count = end - begin;
        int stage = 0;
        uint32_t phase = 0;
        for (uint32_t j = 0; j < count; ++j) {
            const uint32_t tile = begin + j, slots = min(kQpKeys, seen - tile * kQpKeys);
            if (!warp_waited(&raw_full[stage], phase)) { gave_up(kErrFullWaitTimeout); break; }
            const uint8_t* const raw = raw_smem + stage * kQpRaw<kBlocks>;
            const __half* const scales = reinterpret_cast<const __half*>(raw + 2 * kCodes);
            const int shift = q4_shift(q4_largest_scale<kBlocks, kQpKeys>(scales, slots, lane, [&](uint32_t r, uint32_t) { atomicMin(&bad_key, tile * kQpKeys + r); }));
            if (j > 1 && !warp_waited(&k_free[j & 1], ((j >> 1) - 1) & 1)) { gave_up(kErrEmptyWaitTimeout); break; }
            q4_unpack_tile<kBlocks, kQpKeys, kId>(raw, scales, slots, shift, k_smem + (j & 1) * 2 * kKPlane, id);
            if (id == 0) k_unit[j & 3] = power_of_two(-shift);
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&k_full[j & 1]); mbar_arrive(&raw_free[stage]); }
            if (++stage == kQpStages) { stage = 0; phase ^= 1u; }
        }
    } else if (warp < kQpIssueWarp) {                         // values: the same; the first thread keeps the ring filled, ahead of what the warp has to wait for
        constexpr uint32_t kId = (kQpIssueWarp - kQpValueWarp) * 32;
        const uint32_t id = threadIdx.x - kQpValueWarp * 32, count = end - begin;
        if (id == 0) {
            asm volatile("fence.proxy.async;" ::: "memory");      // the stores of the launch before come ahead of the copies
            for (uint32_t j = 0; j < min(count, kQpStages - 1u); ++j) bring(begin + j, j);
        }
        __syncwarp();
        int stage = 0;
        uint32_t phase = 0, j = 0, brought = min(count, kQpStages - 1u);
        for (; j < count; ++j) {
            const uint32_t tile = begin + j, slots = min(kQpKeys, seen - tile * kQpKeys);
            if (!warp_waited(&raw_full[stage], phase)) { gave_up(kErrFullWaitTimeout); break; }
            const uint8_t* const raw = raw_smem + stage * kQpRaw<kBlocks>;
            const __half* const scales = reinterpret_cast<const __half*>(raw + 2 * kCodes + kScales);
            const int shift = q4_shift(q4_largest_scale<kBlocks, kQpKeys>(scales, slots, lane, [&](uint32_t r, uint32_t block) { atomicMin(&bad_value[block], tile * kQpKeys + r); }));
            if (j > 1 && !warp_waited(&v_free[j & 1], ((j >> 1) - 1) & 1)) { gave_up(kErrEmptyWaitTimeout); break; }
            q4_unpack_tile<kBlocks, kQpKeys, kId>(raw + kCodes, scales, slots, shift, v_smem + (j & 1) * 2 * kKPlane, id);
            if (id == 0) v_unit[j & 3] = power_of_two(-shift) * (1.0f / 16384.0f);      // a weight of 1 is 2^14
            async_proxy_fence();
            __syncwarp();
            if (lane == 0) { mbar_arrive(&v_full[j & 1]); mbar_arrive(&raw_free[stage]); }
            if (id == 0 && j + kQpStages - 1 < count) {           // the stage of the tile before, once the values' warps are done with it as well
                const uint32_t to_stage = (j + kQpStages - 1) % kQpStages;
                if (j == 0 || mbar_wait(&raw_free[to_stage], ((j - 1) / kQpStages) & 1u)) {
                    bring(tile + kQpStages - 1, to_stage);
                    ++brought;
                } else {
                    atomicExch(p.error_word, kErrEmptyWaitTimeout);       // the waits for the tile run out as well
                }
            }
            __syncwarp();
            if (++stage == kQpStages) { stage = 0; phase ^= 1u; }
        }
        if (id == 0)                                              // given up: what is under way lands before the memory is another's
            for (; j < brought; ++j) mbar_wait(&raw_full[j % kQpStages], (j / kQpStages) & 1u);
    } else {                                                  // the tensor cores
        constexpr uint32_t score_desc = umma_idesc_f16(kQpRows, kQpKeys), out_desc = umma_idesc_f16(kQpRows, kDim, true), kSteps = kDim / 16;
        const uint64_t k_desc = umma_desc_k_sw128(smem_u32(k_smem)), v_desc = umma_desc_mn_sw128(smem_u32(v_smem), kKPlane / kHalves);
        // a descriptor's start address counts 16-byte units: 16 dimensions are two of them, 16 slots of values 128
        auto scores = [&](uint32_t b) {
            tc_fence_after_sync();
            if (elected()) {
#pragma unroll
                for (int c = 0; c < 3; ++c) {                     // lower times upper, upper times lower, upper times upper
                    const uint32_t qp = c == 0 ? 1 : 0, kp = c == 1 ? 1 : 0;
#pragma unroll
                    for (uint32_t k = 0; k < kSteps; ++k)
                        tc_mma_f16_ts(tmem + kQpScores + k % kQpShares * kQpKeys, tmem + kQpQ + qp * (kDim / 2) + 8 * k,
                                      k_desc + (((b * 2 + kp) * kKPlane + (k / 4) * (kKPlane / kHalves)) >> 4) + 2 * (k % 4), score_desc, c > 0 || k >= kQpShares);
                }
                tc_commit(&k_free[b]);
                tc_commit(&s_full);
            }
            __syncwarp();
        };
        bool ok = warp_waited(&q_full, 0) && warp_waited(&k_full[0], 0);
        if (ok) scores(0);
        const uint32_t count = end - begin;
        for (uint32_t j = 0; ok && j < count; ++j) {
            if (j + 1 < count) {
                ok = warp_waited(&k_full[(j + 1) & 1], ((j + 1) >> 1) & 1) && warp_waited(&s_empty, j & 1);
                if (!ok) break;
                scores((j + 1) & 1);
            }
            ok = warp_waited(&v_full[j & 1], (j >> 1) & 1) && warp_waited(&p_full, j & 1) && (j == 0 || warp_waited(&o_empty, (j - 1) & 1));
            if (!ok) break;
            tc_fence_after_sync();
            if (elected()) {
#pragma unroll
                for (int c = 0; c < 3; ++c) {
                    const uint32_t pp = c == 0 ? 1 : 0, vp = c == 1 ? 1 : 0;
#pragma unroll
                    for (uint32_t k = 0; k < kQpKeys / 16; ++k)
                        tc_mma_f16_ts(tmem + kQpOut, tmem + kQpP + 32 * pp + 8 * k, v_desc + (((j & 1) * 2 + vp) * kKPlane >> 4) + 128 * k, out_desc, (c | k) > 0);
                }
                tc_commit(&v_free[j & 1]);
                tc_commit(&o_full);
            }
            __syncwarp();
        }
        if (!ok) gave_up(kErrFullWaitTimeout);
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kQpIssueWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, kQpColumns);
    }
}

}  // namespace zk
