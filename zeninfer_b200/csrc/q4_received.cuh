// What the slots of a cache in 4 bits received from a block of many rows, heads of 64 or 128 values, on the tensor cores (tcgen05).
//
// received_j = sum over rows r that see slot j of exp2(s_rj - e_r), e_r = m_r + log2 l_r: only known when the rows are done, so the scores are formed a second time, the
// operands and the three products those of q4_prompt.cuh, which left its queries in the operand's layout.  Here the slots are the matrix's rows: a thread owns a slot and adds
// up over the columns, in a fixed order, without exchanges.
//
// A CTA keeps 128 or 256 slots unpacked in shared memory and walks the tiles of 128 rows; a stage of its ring is 64 dimensions of a tile's two parts.  With 256 slots a
// tile that comes out of L2 serves two matrices, which alternate between the accumulators' two buffers: 16 warps exponentiate one while the other is formed.  Each 64
// dimensions have an accumulator of their own, corrections first.  Two warps issue the products, a unit each in turn: what one spends on waits and commits the other fills, for
// the tensor cores take an instruction only when they are done with the one before.  Bounded by the shared memory: a product of 128 x 128 x 16 reads 8 KB there (64 cycles, what it takes
// on the tensor cores), and the copies and the rows' factors need the rest of some 95 cycles.  512 tokens at 8192 slots of 8 kv heads of 128: 105 us, 0.6 of the rate three products could
// have; 131 with 128 slots a CTA, 381 with mma.sync.
#pragma once
#include "q4_prompt.cuh"

namespace zk {

constexpr uint32_t kQrSlots = 128, kQrStages = 3, kQrSumWarps = 16, kQrIssueWarp = 16, kQrCopyWarp = 18, kQrThreads = 19 * 32, kQrSets = 2;
template <int kBlocks> constexpr uint32_t kQrPlane = kQrSlots * kBlocks * 64;
constexpr uint32_t kQrChunk = kQpRows * 128;                  // bytes: a part of 64 dimensions of a tile of rows
template <int kBlocks> constexpr uint32_t q4_received_smem(uint32_t sets) { return 1024 + sets * 2 * kQrPlane<kBlocks> + kQrStages * 2 * kQrChunk; }

// grid = (runs of sets * 128 slots, kv_heads)
template <int kBlocks>
__global__ void __launch_bounds__(kQrThreads, 1) q4_received_kernel(const __grid_constant__ Q4Attend p, uint32_t sets) {
    constexpr uint32_t kHalves = kBlocks / 2, kPlane = kQrPlane<kBlocks>, kScores = kHalves * kQpRows;
    extern __shared__ uint8_t qr_smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(qr_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t* const k_smem = smem;                             // [set][plane][64 dimensions][128 slots][128 bytes]
    uint8_t* const q_smem = k_smem + sets * 2 * kPlane;       // [stage][plane][128 rows][128 bytes]
    __shared__ __align__(16) float2 of_row[kQpRows];                        // what makes scores of a row's products; its e
    __shared__ uint64_t q_full[kQrStages], q_free[kQrStages], s_full[2], s_free[2];
    __shared__ uint32_t tmem_slot;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, h = blockIdx.y, rows = p.tokens * p.group, row_tiles = (rows + kQpRows - 1) / kQpRows;
    const uint32_t cta_slot = blockIdx.x * sets * kQrSlots;
    if (threadIdx.x == 0) {
        for (uint32_t b = 0; b < kQrStages; ++b) { mbar_init(&q_full[b], 1); mbar_init(&q_free[b], sets); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(&s_full[b], 1); mbar_init(&s_free[b], kQrSumWarps); }
        mbar_fence_init();
    }
    pdl_launch_dependents();
    pdl_wait();
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) return;
    const uint32_t filled = filled_in, seen = filled + p.tokens;
    if (cta_slot >= seen) return;
    if (warp == kQrIssueWarp) tmem_alloc(&tmem_slot, 512);
    const uint32_t slots = min(sets * kQrSlots, seen - cta_slot);
    const size_t first_slot = static_cast<size_t>(h) * p.cache.slots + cta_slot;
    uint32_t top = 0;
    for (uint32_t m = 0; m * kQrSlots < slots; ++m)
        top = max(top, q4_largest_scale<kBlocks, kQrSlots>(p.cache.k_scales + (first_slot + m * kQrSlots) * kBlocks, slots - m * kQrSlots, lane, [](uint32_t, uint32_t) {}));
    const int shift = q4_shift(top);
    for (uint32_t m = 0; m < sets; ++m) {
        const size_t at = first_slot + m * kQrSlots;
        q4_unpack_tile<kBlocks, kQrSlots, kQrThreads>(p.cache.k_codes + at * (kBlocks * 16), p.cache.k_scales + at * kBlocks, slots > m * kQrSlots ? slots - m * kQrSlots : 0u, shift,
                                                      k_smem + m * 2 * kPlane, threadIdx.x);
    }
    async_proxy_fence();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = tmem_slot;
    // the tiles of rows that see the CTA's first slot; a unit is a tile against a set of slots
    const uint32_t first_tile = cta_slot < filled ? 0u : (cta_slot - filled) * p.group / kQpRows, units = (row_tiles - first_tile) * sets;
    auto gave_up = [&](int code) { if (lane == 0) atomicExch(p.error_word, code); };

    // A wait that runs out ends its role's loop, and the others' follow.  The summing warps meet here; true where one of them has given up
    auto meet = [&](bool failed) {
        uint32_t any;
        asm volatile("{ .reg .pred p, q; setp.ne.u32 q, %2, 0; barrier.red.or.pred p, 1, %1, q; selp.u32 %0, 1, 0, p; }"
                     : "=r"(any) : "n"(kQrSumWarps * 32), "r"(static_cast<uint32_t>(failed)) : "memory");
        return any != 0;
    };
    if (warp < kQrSumWarps) {                                 // a thread: a slot of each set, 32 columns of every tile
        const uint32_t quad = warp & 3u, part = warp >> 2;
        float sum[kQrSets] = {};
        const float unit = power_of_two(-shift);
        // what a tile's row has, asked for a tile ahead; rows that are none: weights of zero
        auto ask = [&](uint32_t tile) {
            float2 its = make_float2(0.0f, INFINITY);
            if (tile < row_tiles && threadIdx.x < kQpRows && tile * kQpRows + threadIdx.x < rows) {
                its.x = __ldcg(p.factors + (static_cast<size_t>(h) * row_tiles + tile) * kQpRows + threadIdx.x);
                its.y = __ldcg(p.stats + static_cast<size_t>(h) * rows + tile * kQpRows + threadIdx.x);
            }
            return its;
        };
        float2 next = ask(first_tile);
        bool ok = true;
        for (uint32_t u = 0; u < units; ++u) {
            const uint32_t tile = first_tile + u / sets, set = u % sets, b = u & 1u, row0 = tile * kQpRows;
            if (set == 0) {
                if (meet(!ok)) { ok = false; break; }         // the tile before is done with the place
                if (threadIdx.x < kQpRows) of_row[threadIdx.x] = make_float2(next.x * unit, next.y);
                next = ask(tile + 1);
                meet(false);
            }
            ok = ok && warp_waited(&s_full[b], (u >> 1) & 1u);
            if (ok) {
                tc_fence_after_sync();
                const uint32_t slot = cta_slot + set * kQrSlots + quad * 32 + lane, from = tmem + b * kScores + part * 32 + ((quad * 32) << 16);
                // the columns from here on see the slot
                const uint32_t sees = slot < filled ? 0u : (slot - filled) * p.group, column0 = row0 + part * 32;
                float added[4] = {};
                uint32_t share[2][kHalves][16];
                auto load = [&](int c) {
#pragma unroll
                    for (uint32_t i = 0; i < kHalves; ++i) tmem_ld_32x16(from + i * kQpRows + 16 * c, share[c][i]);
                };
                auto add = [&](int c, auto all) {
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float4 two = reinterpret_cast<const float4*>(of_row)[(part * 32 + 16 * c + i) / 2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float s = __uint_as_float(share[c][0][i + e]);
                            if (kHalves > 1) s += __uint_as_float(share[c][kHalves - 1][i + e]);
                            const float w = exp2_fast(e ? fmaf(s, two.z, -two.w) : fmaf(s, two.x, -two.y));
                            if (decltype(all)::value || column0 + 16 * c + i + e >= sees) added[(i + e) & 3] += w;
                        }
                    }
                };
                auto work = [&](auto all) {
                    load(0);
                    tmem_ld_wait();
                    load(1);
                    add(0, all);
                    tmem_ld_wait();
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[b]);
                    add(1, all);
                };
                if (__all_sync(0xffffffffu, sees <= column0)) work(std::true_type{});
                else work(std::false_type{});
                const float both = (added[0] + added[1]) + (added[2] + added[3]);
                if (set == 0) sum[0] += both;
                else sum[1] += both;
            }
        }
        const bool failed = meet(!ok);                        // every warp comes here, those that have given up too
        if (failed) gave_up(kErrTmemWaitTimeout);
        float* const share = reinterpret_cast<float*>(of_row);         // [2 sets][128]: each part adds its own in turn
        for (uint32_t from = 0; from < 4; ++from) {
            if (part == from)
                for (uint32_t m = 0; m < kQrSets; ++m) share[m * kQrSlots + quad * 32 + lane] = (from ? share[m * kQrSlots + quad * 32 + lane] : 0.0f) + sum[m];
            meet(false);
        }
        const uint32_t slot = cta_slot + threadIdx.x;
        if (!failed && threadIdx.x < slots) {
            const size_t at = static_cast<size_t>(h) * p.cache.slots + slot;
            p.weight_out[at] = share[threadIdx.x] + (slot < filled ? p.weight_in[at] : 0.0f);
        }
    } else if (warp < kQrCopyWarp) {
        constexpr uint32_t desc = umma_idesc_f16(kQrSlots, kQpRows);
        const uint32_t b = warp - kQrIssueWarp;               // the accumulators' buffer: units b, b + 2, ..
        const uint64_t k_desc = umma_desc_k_sw128(smem_u32(k_smem)), q_desc = umma_desc_k_sw128(smem_u32(q_smem));
        bool ok = true;
        for (uint32_t u = b; ok && u < units; u += 2) {
            const uint32_t set = u % sets;
            ok = u < 2 || warp_waited(&s_free[b], ((u >> 1) - 1) & 1u);
            for (uint32_t c = 0; ok && c < kHalves; ++c) {
                const uint32_t chunk = u / sets * kHalves + c, stage = chunk % kQrStages;
                ok = warp_waited(&q_full[stage], (chunk / kQrStages) & 1u);
                if (!ok) break;
                tc_fence_after_sync();
                const uint64_t k_at = k_desc + ((set * 2 * kPlane + c * (kPlane / kHalves)) >> 4), q_at = q_desc + (stage * 2 * kQrChunk >> 4);
                if (elected()) {
#pragma unroll
                    for (uint32_t i = 0; i < 3; ++i) {        // lower times upper, upper times lower, upper times upper
                        const uint32_t kp = i == 0 ? 1 : 0, qp = i == 1 ? 1 : 0;
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                            tc_mma_f16(tmem + b * kScores + c * kQpRows, k_at + (kp * kPlane >> 4) + 2 * k, q_at + (qp * kQrChunk >> 4) + 2 * k, desc, (i | k) > 0);
                    }
                    tc_commit(&q_free[stage]);
                    if (c + 1 == kHalves) tc_commit(&s_full[b]);
                }
                __syncwarp();
            }
        }
        if (!ok) gave_up(kErrFullWaitTimeout);
    } else if (lane == 0) {                                   // copies, a stage each 64 dimensions of a tile
        const uint32_t count = (row_tiles - first_tile) * kHalves;
        const uint8_t* const from = reinterpret_cast<const uint8_t*>(p.queries) + (static_cast<size_t>(h) * row_tiles + first_tile) * 2 * kQpQPlane<kBlocks>;
        asm volatile("fence.proxy.async;" ::: "memory");      // the stores of the launch before come ahead of the copies
        bool ok = true;
        uint32_t j = 0;
        for (; j < count; ++j) {
            const uint32_t stage = j % kQrStages;
            if (j >= kQrStages && !(ok = mbar_wait(&q_free[stage], (j / kQrStages - 1) & 1u))) break;
            mbar_arrive_expect_tx(&q_full[stage], 2 * kQrChunk);
            for (uint32_t plane = 0; plane < 2; ++plane)
                bulk_g2s(q_smem + (stage * 2 + plane) * kQrChunk, from + static_cast<size_t>(j / kHalves) * 2 * kQpQPlane<kBlocks> + plane * kQpQPlane<kBlocks> + j % kHalves * kQrChunk, kQrChunk,
                         &q_full[stage]);
        }
        if (!ok) atomicExch(p.error_word, kErrEmptyWaitTimeout);
        for (uint32_t i = j - min(j, kQrStages); i < j; ++i) mbar_wait(&q_full[i % kQrStages], (i / kQrStages) & 1u);      // what is under way lands before the memory is another's
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    if (warp == kQrIssueWarp) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace zk
