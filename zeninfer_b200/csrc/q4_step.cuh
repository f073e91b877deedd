// Attention of up to four rows a kv head over a cache held in 4 bits (a step of a model whose groups are of one to four query heads): one launch that
// appends, attends and, for caches of moderate size, ends the call.
//
// The arithmetic is q4_attention.cuh's; a column of the products is a digit of a row, so that four rows fill the eight columns.  What is different is
// what a step's time is made of: round trips to memory and launches.  So a CTA lays out the rows of queries itself while its first tiles are on
// their way; the warp that has the tile of a new slot quantises it, writes it to the cache and into the tile when that has landed.
//   kCluster    the CTAs of a kv head are a cluster (up to eight): their sums meet through distributed shared memory, the scores stay in shared memory, and what the
//               slots received is added before the launch ends
//   else        runs of slots on all SMs; q4_finish_kernel puts them together
// What bounds it: round trips and two cluster barriers up to some thousand slots (5.7 us at 20 slots of 2 kv heads of 64, 8.6 at 1000 of 8 of 128 with weights, of which a launch is 3); beyond,
// the instructions of the tiles' loop, where warps wait for the ALU pipe and for one another, and the ends of the launch around it (29.5 us at 65501 slots, 2.6 TB/s of codes and scales; the
// bytes alone would be 11.6.  Over the whole launch 56 % of the issue slots and 53 % of the ALU pipe are used).  Which of the two is taken goes by the cache's size, for what is filled is
// known on the device only: 1000 filled slots take 8.6 us in a cache of 8192 and 11.7 in one of 32768.
#pragma once
#include <cooperative_groups.h>

#include "q4_attention.cuh"

namespace zk {

constexpr uint32_t kQ4ClusterTiles = 4;      // tiles of a warp at most, in a cluster
constexpr int kQ4StepWarps = 8;

// Dynamic shared memory: the warps' rings, the queries, and (a cluster that adds up weights) the warps' scores [tile][row][slot].
template <int kBlocks>
__host__ __device__ constexpr uint32_t q4_step_smem(bool keep_scores) {
    return kQ4StepWarps * kQ4Stages * q4_stage_bytes<kBlocks>() + kBlocks * 512 + (keep_scores ? kQ4StepWarps * kQ4ClusterTiles * 4 * kQ4Tile * 4 : 0);
}

// grid = (splits, 1, kv_heads); kCluster: a cluster of `splits`
template <int kBlocks, bool kCluster>
__global__ void __launch_bounds__(kQ4StepWarps * 32, kBlocks > 4 ? 1 : 2) q4_step_kernel(const __grid_constant__ Q4Attend p) {
    namespace cg = cooperative_groups;
    constexpr int kWarps = kQ4StepWarps, kDim = kBlocks * 32;
    constexpr uint32_t kStage = q4_stage_bytes<kBlocks>(), kCodes = kQ4Tile * kBlocks * 16, kScales = kQ4Tile * kBlocks * 2, kPieces = 2 * kBlocks;
    constexpr uint32_t kPitch = kDim + 8;                         // of a row of a warp's sums: a quad's rows eight banks apart
    extern __shared__ __align__(128) uint8_t q4_smem[];
    __shared__ uint64_t landed[kWarps][kQ4Stages];
    __shared__ float row_max[kWarps][4], row_sum[kWarps][4], row_unit[kWarps], row_factor[4];
    __shared__ __align__(16) uint4 fresh_codes[4][kPieces];       // the new slots this CTA has: blocks of the key, then of the value
    __shared__ __half fresh_scales[4][kPieces];
    __shared__ float cta_out[4 * kDim];                           // read by the cluster
    __shared__ float2 cta_stats[4];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, t = lane & 3u, h = blockIdx.z, rows = p.tokens * p.group;
    uint4* const queries = reinterpret_cast<uint4*>(q4_smem + kWarps * kQ4Stages * kStage);
    float* const kept = reinterpret_cast<float*>(queries + kBlocks * 32) + warp * kQ4ClusterTiles * 4 * kQ4Tile;
    if (lane == 0) {
        for (int s = 0; s < kQ4Stages; ++s) mbar_init(&landed[warp][s], 1);
        mbar_fence_init();
    }
    __syncwarp();
    pdl_launch_dependents();
    pdl_wait();
    // what does not depend on the place is asked for beside it: the warp's row of queries, and its block of the first new slot
    Q4Raw raw[kBlocks], raw_fresh;
    const uint32_t own_item = warp >= 4 ? warp - 4 : kPieces;
    if (warp < rows) {
        const float* from = p.q + (warp / p.group) * p.q_ld + static_cast<size_t>(h * p.group + warp % p.group) * kDim;
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) raw[g] = q4_raw(from, g * 32 + lane, p.turn);
    }
    const float* const new_k = p.k + static_cast<size_t>(h) * kDim;
    const float* const new_v = p.v + static_cast<size_t>(h) * kDim;
    auto fresh_raw = [&](uint32_t token, uint32_t item) {
        return item >= kBlocks ? Q4Raw{__ldcg(new_v + token * p.kv_ld + (item - kBlocks) * 32 + lane), 0.0f} : q4_raw(new_k + token * p.kv_ld, item * 32 + lane, p.turn);
    };
    if (own_item < kPieces) raw_fresh = fresh_raw(0, own_item);
    const int filled_in = *reinterpret_cast<const volatile int*>(p.filled);
    const int position = p.turn.pairs ? *reinterpret_cast<const volatile int*>(p.position) : 0;
    if (!q4_places_ok(filled_in, position, p.tokens, p.cache.slots, p.turn.pairs, p.turn.positions)) {       // all CTAs alike
        if (threadIdx.x == 0 && blockIdx.x == 0 && h == 0) atomicExch(p.error_word, kErrBadPosition);
        return;
    }
    const uint32_t filled = filled_in, seen = filled + p.tokens;
    const Q4Runs runs = q4_runs(seen, p.splits, kWarps, kQ4Tile);
    const uint32_t begin = blockIdx.x * runs.per, end = min(runs.tiles, begin + runs.per);
    if (!kCluster && begin >= end) return;                                                // nobody counts on this run
    uint8_t* ring = q4_smem + warp * kQ4Stages * kStage;
    const size_t head_slots = static_cast<size_t>(h) * p.cache.slots;
    auto fetch = [&](uint32_t tile, int stage) {
        const size_t slot = head_slots + static_cast<size_t>(tile) * kQ4Tile;
        uint8_t* to = ring + stage * kStage;
        mbar_arrive_expect_tx(&landed[warp][stage], kStage);
        bulk_g2s(to, p.cache.k_codes + slot * (kBlocks * 16), kCodes, &landed[warp][stage]);
        bulk_g2s(to + 2 * kCodes, p.cache.k_scales + slot * kBlocks, kScales, &landed[warp][stage]);
        bulk_g2s(to + kCodes, p.cache.v_codes + slot * (kBlocks * 16), kCodes, &landed[warp][stage]);
        bulk_g2s(to + 2 * kCodes + kScales, p.cache.v_scales + slot * kBlocks, kScales, &landed[warp][stage]);
    };
    const uint32_t mine = begin + warp < end ? (end - begin - warp + kWarps - 1) / kWarps : 0u;      // tiles of this warp
    if (lane == 0) {
        asm volatile("fence.proxy.async;" ::: "memory");       // the stores of earlier launches come ahead of the copies
        for (uint32_t i = 0; i < min(mine, static_cast<uint32_t>(kQ4Stages)); ++i) fetch(begin + warp + i * kWarps, i);
    }
    // the rows, rotated and laid out, by warps 0 .. 3; zeros where there are fewer.  Warps 4 .. 7 quantise the blocks of new slots that lie in this CTA's tiles.
    float x[kBlocks] = {};
    if (warp < rows) {
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) x[g] = q4_rotated(raw[g], g * 32 + lane, p.turn, static_cast<size_t>(position) + warp / p.group);
    }
    for (uint32_t token = 0; token < p.tokens; ++token) {
        const uint32_t tile = (filled + token) / kQ4Tile;
        if (tile < begin || tile >= end) continue;
        for (uint32_t item = own_item; item < kPieces; item += 4) {
            const Q4Raw its = token == 0 && item == own_item ? raw_fresh : fresh_raw(token, item);
            const float value = item >= kBlocks ? its.mine : q4_rotated(its, item * 32 + lane, p.turn, static_cast<size_t>(position) + token);
            __half scale;
            const uint8_t byte = q4_append_block<kBlocks>(p, value, h, token, item, filled, lane, scale);
            if (lane < 16) reinterpret_cast<uint8_t*>(&fresh_codes[token][item])[lane] = byte;
            if (lane == 0) fresh_scales[token][item] = scale;
        }
    }
    if (warp < 4) {
        const float factor = q4_lay_row<kBlocks, true>(x, queries, warp, p.scale, lane);
        if (lane == 0) row_factor[warp] = factor;
    }
    __syncthreads();
    const uint32_t last_seen = filled + min(t, rows - 1) / p.group, least = filled;      // of the lane's row, of all rows
    const float factor = row_factor[t];
    const float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    uint4 own_query[kBlocks];
#pragma unroll
    for (int g = 0; g < kBlocks; ++g) own_query[g] = queries[g * 32 + lane];
    float acc[2 * kBlocks][4] = {};
    float m = -INFINITY, l = 0.0f;
    // Weights times 2^(kFull - unit) times their slot's d are below 2^14: d is below 2^unit and a weight at most 2^kSlack.
    constexpr float kSlack = 8.0f;
    constexpr int kFull = 6, kHeadroom = 14;            // f16's exponent field less 14: the power of two above a scale
    int unit = -32;

    // A tile; kWhole: every row sees every slot of it.
    auto work = [&](const uint8_t* stage, uint32_t slot0, uint32_t turn, auto whole) {
        constexpr bool kWhole = decltype(whole)::value;
        const uint32_t a = lane >> 2;                     // the lane's slots are a, a + 8, a + 16, a + 24, its row is t
        const __half* k_scales = reinterpret_cast<const __half*>(stage + 2 * kCodes);
        const __half* v_scales = k_scales + kQ4Tile * kBlocks;
        const uint32_t matrix = ((lane >> 3) * kBlocks * 8 + (lane & 7u)) * 16;
        float s[4] = {};                                  // slot a + 8 i
        {
            Q4Scales<kBlocks> d;
            d.load(k_scales, a);
            uint32_t w[kBlocks][4];
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) ldmatrix_x4(w[g], smem_u32(stage) + matrix + g * 128);      // all at once: they are not moved past one another
#pragma unroll
            for (int g = 0; g < kBlocks; ++g) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t u = w[g][2 * half], v = w[g][2 * half + 1], x = u >> 8, y = v >> 8;
                    // with their offset taken off: sums of codes as they stand are far from zero, and what the products cut off was a score's last 4 bits
                    const uint32_t even[4] = {signed_low(u), signed_low(v), signed_high(u), signed_high(v)};
                    const uint32_t odd[4] = {signed_low(x), signed_low(y), signed_high(x), signed_high(y)};
                    float c[4];
                    mma_f16(c, even, own_query[g].x, own_query[g].y, zero);
                    mma_f16(c, odd, own_query[g].z, own_query[g].w, c);
                    s[2 * half] = fmaf(d.of(2 * half, g), c[0] + c[1], s[2 * half]);
                    s[2 * half + 1] = fmaf(d.of(2 * half + 1, g), c[2] + c[3], s[2 * half + 1]);
                }
            }
        }
        uint32_t values[kBlocks][4];
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) ldmatrix_x4_trans(values[g], smem_u32(stage) + kCodes + matrix + g * 128);
        auto hidden = [&](int i) { return !kWhole && slot0 + 8 * i + a > last_seen; };
        // the largest scale of a value that any row sees, as a power of two
        const uint32_t top = __reduce_max_sync(0xffffffffu, kWhole || slot0 + lane < seen ? Q4Scales<kBlocks>::largest(v_scales, lane) : 0u);
        const int new_unit = max(unit, min(static_cast<int>(top >> 10), 30) - kHeadroom);
        if constexpr (!kWhole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = hidden(i) ? -INFINITY : s[i];
        }
        float x = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16)) * factor;
        const float next = x > m + kSlack ? x : m;        // a maximum that is little larger leaves the weights above one, and the sums as they are
        if (kCluster ? p.weight_out != nullptr : p.scores != nullptr) {
            if (kCluster || t < rows) {
                float* to = kCluster ? kept + (turn * 4 + t) * kQ4Tile + a : p.scores + (static_cast<size_t>(h) * rows + t) * p.cache.slots + slot0 + a;
#pragma unroll
                for (int i = 0; i < 4; ++i) to[8 * i] = s[i] * factor;
            }
        }
        if (__any_sync(0xffffffffu, next != m || new_unit != unit)) {
            const float corr = m == -INFINITY ? 0.0f : exp2_fast(m - next);
            l *= corr;
            m = next;
            const float by = unit == -32 ? 0.0f : corr * power_of_two(unit - new_unit);
#pragma unroll
            for (int j = 0; j < 2 * kBlocks; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] *= by;
            unit = new_unit;
        }
        const float up = power_of_two(kFull - unit), from = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float w = exp2_fast(fmaf(s[i], factor, -from));
            l += w;
            s[i] = w * up;
        }
        Q4Scales<kBlocks> d;
        d.load(v_scales, a);
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            float sum[2][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t u = values[g][2 * half], v = values[g][2 * half + 1], x = u >> 8, y = v >> 8;
                // dimensions 2r and 16 + 2r, 2r + 1 and 17 + 2r of the block, r the lane's row of the operand
                const uint32_t even[4] = {signed_low(u), signed_high(u), signed_low(v), signed_high(v)};
                const uint32_t odd[4] = {signed_low(x), signed_high(x), signed_low(y), signed_high(y)};
                // a slot that is not seen may hold anything
                const float wa = hidden(2 * half) ? 0.0f : s[2 * half] * d.of(2 * half, g), wb = hidden(2 * half + 1) ? 0.0f : s[2 * half + 1] * d.of(2 * half + 1, g);
                const float ha = upper_digit(wa), hb = upper_digit(wb);
                const uint32_t b0 = transposed(pack_f16(ha, wa - ha)), b1 = transposed(pack_f16(hb, wb - hb));
                mma_f16(sum[0], even, b0, b1, half ? static_cast<const float (&)[4]>(sum[0]) : zero);
                mma_f16(sum[1], odd, b0, b1, half ? static_cast<const float (&)[4]>(sum[1]) : zero);
            }
            add_pairs(acc[2 * g], sum[0]);
            add_pairs(acc[2 * g + 1], sum[1]);
        }
    };

    bool failed = false;
    int stage = 0;
    uint32_t phase = 0;
    for (uint32_t i = 0; i < mine; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait(&landed[warp][stage], phase))) {
            // the copies that are under way land (or are given up) before the ring is used for anything else
            if (lane == 0) {
                atomicExch(p.error_word, kErrFullWaitTimeout);
                for (uint32_t j = i; j < min(mine, i + kQ4Stages); ++j) mbar_wait(&landed[warp][j % kQ4Stages], (j / kQ4Stages) & 1u);
            }
            __syncwarp();
            failed = true;
            break;
        }
        const uint32_t tile = begin + warp + i * kWarps, slot0 = tile * kQ4Tile;
        uint8_t* const at = ring + stage * kStage;
        if (slot0 + kQ4Tile > filled) {           // new slots into the tile, which came without them
            for (uint32_t token = 0; token < p.tokens; ++token) {
                const uint32_t slot = filled + token - slot0;                  // in the tile where it is below 32
                if (slot >= kQ4Tile || lane >= kPieces) continue;
                const uint32_t value = lane >= kBlocks, block = value ? lane - kBlocks : lane;
                *reinterpret_cast<uint4*>(at + value * kCodes + (((slot >> 3) * kBlocks + block) * 8 + (slot & 7u)) * 16) = fresh_codes[token][lane];
                reinterpret_cast<__half*>(at + 2 * kCodes + value * kScales)[slot * kBlocks + block] = fresh_scales[token][lane];
            }
            __syncwarp();
        }
        if (slot0 + kQ4Tile - 1 <= least) work(at, slot0, i, std::true_type{});
        else work(at, slot0, i, std::false_type{});
        __syncwarp();                       // everybody is done with the stage
        if (lane == 0 && i + kQ4Stages < mine) fetch(tile + kQ4Stages * kWarps, stage);
        if (++stage == kQ4Stages) {
            stage = 0;
            phase ^= 1u;
        }
    }

    // the warp's sums into its ring's memory, [row][dimension]
    float* sums = reinterpret_cast<float*>(ring);
    l += __shfl_xor_sync(0xffffffffu, l, 4);
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    l += __shfl_xor_sync(0xffffffffu, l, 16);
    if (lane < 4) { row_max[warp][t] = m; row_sum[warp][t] = failed ? NAN : l; }
#pragma unroll
    for (int g = 0; g < kBlocks; ++g) {
        const float (&c)[4] = acc[2 * g];
        const float (&d)[4] = acc[2 * g + 1];
        float2* to = reinterpret_cast<float2*>(sums + t * kPitch + g * 32) + (lane >> 2);
        to[0] = make_float2(c[0] + c[1], d[0] + d[1]);
        to[8] = make_float2(c[2] + c[3], d[2] + d[3]);
    }
    if (lane == 0) row_unit[warp] = unit == -32 ? 0.0f : power_of_two(unit - kFull);
    __syncthreads();
    // the warps' shares of the rows: lane w * 4 + r of every warp has what warp w's sums of row r count
    auto over_groups_of_four = [](float x, auto op) {
        x = op(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = op(x, __shfl_xor_sync(0xffffffffu, x, 8));
        return op(x, __shfl_xor_sync(0xffffffffu, x, 16));
    };
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto added = [](float x, float y) { return x + y; };
    float weight_before[kQ4ClusterTiles] = {};
    if (kCluster && p.weight_out) {
#pragma unroll
        for (uint32_t i = 0; i < kQ4ClusterTiles; ++i) {
            const uint32_t slot = (begin + warp + i * kWarps) * kQ4Tile + lane;
            if (i < mine && slot < filled) weight_before[i] = __ldcg(p.weight_in + head_slots + slot);
        }
    }
    {
        const float its = row_max[lane >> 2][t], top = over_groups_of_four(its, larger);
        const float by = its == -INFINITY ? 0.0f : exp2_fast(its - top), by_unit = by * row_unit[lane >> 2];
        const float sum = over_groups_of_four(its == -INFINITY ? row_sum[lane >> 2][t] : by * row_sum[lane >> 2][t], added);      // no maximum: none, or what is not a number
        for (uint32_t i = threadIdx.x; i < rows * kDim; i += kWarps * 32) {
            const uint32_t r = i / kDim;                       // the same for all of a warp
            float o = 0.0f, part[kWarps];
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) part[w] = reinterpret_cast<const float*>(q4_smem + w * kQ4Stages * kStage)[r * kPitch + i % kDim];
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) o += __shfl_sync(0xffffffffu, by_unit, w * 4 + r) * part[w];
            if (kCluster) cta_out[i] = o;
            else p.part_out[((static_cast<size_t>(h) * p.splits + blockIdx.x) * rows + r) * kDim + i % kDim] = o;
        }
        if (warp == 0 && lane < 4) {
            if (kCluster) cta_stats[lane] = make_float2(top, sum);
            else if (lane < rows) reinterpret_cast<float2*>(p.part_stats)[(static_cast<size_t>(h) * p.splits + blockIdx.x) * rows + lane] = make_float2(top, sum);
        }
    }
    if constexpr (kCluster) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        // the CTAs' shares likewise: lane c * 4 + r of every warp has what CTA c's sums of row r count
        const float2 its = (lane >> 2) < p.splits ? *cluster.map_shared_rank(cta_stats + t, lane >> 2) : make_float2(-INFINITY, 0.0f);
        float part[8];
        const uint32_t i = blockIdx.x * (kWarps * 32) + threadIdx.x;          // each CTA has a share of the rows' dimensions
#pragma unroll
        for (uint32_t c = 0; c < 8; ++c) part[c] = c < p.splits && i < rows * kDim ? *cluster.map_shared_rank(cta_out + i, c) : 0.0f;
        const float top = over_groups_of_four(its.x, larger), by = its.x == -INFINITY ? 0.0f : exp2_fast(its.x - top);
        const float sum = over_groups_of_four(its.x == -INFINITY ? its.y : by * its.y, added), share = by / sum;
        if (blockIdx.x == 0 && warp == 0 && lane < rows && (!(sum > 0.0f) || !(sum < INFINITY))) atomicExch(p.error_word, kErrNonFinite);
        auto put = [&](uint32_t at, const float (&of)[8]) {
            const uint32_t r = min(at / kDim, 3u), token = r / p.group, head = h * p.group + r % p.group;
            float o = 0.0f;
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) o += __shfl_sync(0xffffffffu, share, c * 4 + r) * of[c];
            if (at < rows * kDim) p.out[(static_cast<size_t>(token) * p.heads + head) * kDim + at % kDim] = o;
        };
        put(i, part);
        for (uint32_t more = i + p.splits * kWarps * 32; more - threadIdx.x % 32 < rows * kDim; more += p.splits * kWarps * 32) {
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) part[c] = c < p.splits && more < rows * kDim ? *cluster.map_shared_rank(cta_out + more, c) : 0.0f;
            put(more, part);
        }
        if (p.weight_out) {
            const float whole = top + log2f(sum);              // of row t
#pragma unroll
            for (uint32_t j = 0; j < kQ4ClusterTiles; ++j) {
                float received = 0.0f;
#pragma unroll
                for (uint32_t r = 0; r < 4; ++r) {
                    const float of_row = __shfl_sync(0xffffffffu, whole, r);
                    if (r < rows && j < mine) received += exp2_fast(kept[(j * 4 + r) * kQ4Tile + lane] - of_row);      // a slot the row does not see: minus infinity
                }
                const uint32_t slot = (begin + warp + j * kWarps) * kQ4Tile + lane;
                if (j < mine && slot < seen) p.weight_out[head_slots + slot] = received + weight_before[j];
            }
        }
        cluster.sync();                     // nobody leaves while its shared memory is read
    }
}

}  // namespace zk
